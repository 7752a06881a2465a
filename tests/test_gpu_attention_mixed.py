"""GPU: packed calls whose sequences differ by far from their average: a long prompt among single tokens, single tokens on caches of
very different fill.  The bound is that of the batched and packed tests: with u half a step of the type, n keys and A = sum p |v|,
A (u + 2 eta + n 2^-23) + u |o|, eta = (D + 1.5) 2^-23 sum |q k| scale + 4e-6."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from segquant_b200 import ops

DEV = "cuda"


def _check(got, q, k, v, causal):
    tq, hq, d = q.shape
    n, hkv, _ = k.shape
    u = torch.finfo(q.dtype).eps / 2
    q, k, v = (t.double().transpose(0, 1) for t in (q, k, v))
    k, v = k.repeat_interleave(hq // hkv, 0), v.repeat_interleave(hq // hkv, 0)
    s = q @ k.transpose(1, 2) * d ** -0.5
    eta = (d + 1.5) * 2.0 ** -23 * (q.abs() @ k.abs().transpose(1, 2)).amax(dim=-1, keepdim=True) * d ** -0.5 + 4e-6
    if causal:
        s = s.masked_fill(torch.arange(n, device=DEV)[None] > torch.arange(tq, device=DEV)[:, None] + n - tq, -torch.inf)
    p = torch.softmax(s, dim=-1)
    o, a = p @ v, p @ v.abs()
    tol = a * (u + 2 * eta + n * 2.0 ** -23) + u * o.abs() + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    err = (got.double().transpose(0, 1) - o).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("lens,kv_lens,hq,hkv,d", [
    ([1500] + [1] * 120, [1500] + [1 + 37 * i % 900 for i in range(120)], 4, 2, 64),     # few rows a sequence on average
    ([1] * 40 + [700] + [1] * 200, [300] * 40 + [2000] + [5] * 200, 8, 8, 128),
    ([1] * 6, [1, 16000, 33, 9000, 0, 127], 32, 8, 128), ([1] * 3 + [3000], [20, 12000, 1, 3000], 2, 1, 80),
], ids=["prompt_first", "prompt_inside", "uneven_caches", "prompt_last"])
def test_lengths_far_from_their_average(native_lib, lens, kv_lens, hq, hkv, d, dtype):
    g = torch.Generator(device=DEV).manual_seed(9)
    qo, ko = ([0] + torch.tensor(t).cumsum(0).tolist() for t in (lens, kv_lens))
    q = (1.5 * torch.randn(qo[-1], hq, d, generator=g, device=DEV)).to(dtype)
    k, v = (torch.randn(ko[-1], hkv, d, generator=g, device=DEV).to(dtype) for _ in range(2))
    out = ops.attention(q, k, v, causal=True, q_offsets=torch.tensor(qo, dtype=torch.int32, device=DEV),
                        kv_offsets=torch.tensor(ko, dtype=torch.int32, device=DEV))
    for i in range(len(lens)):
        a, b = slice(qo[i], qo[i + 1]), slice(ko[i], ko[i + 1])
        if kv_lens[i] == 0:
            assert not out[a].any()
        else:
            _check(out[a], q[a], k[b], v[b], True)
    assert ops.device_status() == 0
