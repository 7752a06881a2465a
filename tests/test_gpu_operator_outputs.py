"""GPU: outputs that overlap themselves or an input are refused; outputs that only lie between the inputs are not."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from segquant_b200 import ops

DEV = "cuda"


def _x(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device=DEV).to(dtype)


def _refused(calls):
    for i, call in enumerate(calls):
        with pytest.raises(ValueError, match="overlap"):
            call()
            pytest.fail(f"call {i} was not refused")


def test_rotary_outputs(native_lib):
    q, k, pos = _x(2, 8, 4, 64), _x(2, 8, 4, 64), torch.arange(8, device=DEV, dtype=torch.int32)[:, None]
    call = lambda a, b, **kw: ops.rotary(a, b, pos, (64,), **kw)  # noqa: E731
    want = call(q, k)
    one, flat = _x(2, 8, 1, 64).expand(-1, -1, 4, -1), _x(10000)
    long = _x(2, 12, 4, 64)
    _refused([
        lambda: call(q, k, out_q=one), lambda: call(q, k, out_k=one), lambda: call(one, None, out_q=one),          # several heads at one address
        lambda: call(q, None, out_q=flat.as_strided((2, 8, 4, 64), (2048, 256, 32, 1))),                             # heads half over one another
        lambda: call(q, None, out_q=flat.as_strided((2, 8, 4, 64), (512, 64, 64, 1))),                               # a token on the next one's heads
        lambda: call(q, k, out_q=k), lambda: call(q, k, out_k=q), lambda: call(q, k, out_q=k, out_k=k),
        lambda: call(long[:, :8], None, out_q=long[:, 4:]), lambda: call(long[:, 4:], None, out_q=long[:, :8]),       # shifted by tokens
        lambda: call(flat[:4096].view(2, 8, 4, 64), None, out_q=flat[8:4104].view(2, 8, 4, 64)),                       # shifted by columns
    ])
    both = torch.empty_like(q)
    _refused([lambda: call(q, k, out_q=both, out_k=both)])
    # in place, also through another view of the same elements, and outputs between the inputs of one buffer
    a, b = q.clone(), k.clone()
    got = call(a, b, out_q=a.view(2, 8, 4, 64), out_k=b)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[0].data_ptr() == a.data_ptr()
    buf = _x(2, 8, 5, 4, 64)
    buf[:, :, 0], buf[:, :, 1], rest = q, k, buf[:, :, 4].clone()
    call(buf[:, :, 0], buf[:, :, 1], out_q=buf[:, :, 2], out_k=buf[:, :, 3])
    assert torch.equal(buf[:, :, 2], want[0]) and torch.equal(buf[:, :, 3], want[1]) and torch.equal(buf[:, :, 4], rest)
    call(buf[:, :, 0], buf[:, :, 1], out_q=buf[:, :, 0], out_k=buf[:, :, 1])
    assert torch.equal(buf[:, :, 0], want[0]) and torch.equal(buf[:, :, 1], want[1])
    heads = _x(2, 6, 8, 64)                                      # heads first: strides of another order
    out = torch.empty(2, 4, 8, 64, dtype=q.dtype, device=DEV).transpose(1, 2)
    heads[:, :4] = q.transpose(1, 2)
    assert torch.equal(call(heads[:, :4].transpose(1, 2), None, out_q=out)[0], want[0])


def test_attention_outputs(native_lib):
    q, k, v = _x(2, 8, 4, 64), _x(2, 8, 4, 64), _x(2, 8, 4, 64)
    want = ops.attention(q, k, v)
    flat, one = _x(10000), _x(2, 8, 1, 64)
    _refused([
        lambda: ops.attention(q, k, v, out=q), lambda: ops.attention(q, k, v, out=k), lambda: ops.attention(q, k, v, out=v),
        lambda: ops.attention(q, k, v, out=q.view(2, 8, 4, 64)), lambda: ops.attention(q, one, one, out=flat.as_strided((2, 8, 4, 64), (2048, 256, 32, 1))),
        lambda: ops.attention(flat[:4096].view(2, 8, 4, 64), k, v, out=flat[64:4160].view(2, 8, 4, 64)),
        lambda: ops.attention(q, flat[:4096].view(2, 8, 4, 64), v, out=flat[8:4104].view(2, 8, 4, 64)),
    ])
    packed, off = q.view(16, 4, 64), torch.tensor([0, 8, 16], dtype=torch.int32, device=DEV)
    _refused([lambda: ops.attention(packed, packed, packed, q_offsets=off, out=packed)])
    buf = _x(2, 8, 4, 4, 64)                                     # q | k | v | out side by side
    buf[:, :, 0], buf[:, :, 1], buf[:, :, 2] = q, k, v
    ins = buf[:, :, :3].clone()
    ops.attention(buf[:, :, 0], buf[:, :, 1], buf[:, :, 2], out=buf[:, :, 3])
    assert torch.equal(buf[:, :, 3], want) and torch.equal(buf[:, :, :3], ins)
    group = _x(2, 8, 10, 64)                                     # 4 + 1 + 1 heads and the result's 4 in one row
    ops.attention(group[:, :, :4], group[:, :, 4:5], group[:, :, 5:6], out=group[:, :, 6:])
    assert torch.equal(group[:, :, 6:], ops.attention(group[:, :, :4].clone(), group[:, :, 4:5].clone(), group[:, :, 5:6].clone()))
    # few rows, many keys: the joining pass writes behind the one that reads
    q1, kv = _x(1, 1, 4, 64), _x(1, 5000, 4, 64)
    _refused([lambda: ops.attention(q1, kv, kv, out=q1)])
