"""GPU: ops.rotary against the rotation in fp64.

Tolerance, element by element, with u = finfo.eps / 2 of the type (one rounding at the end) and h = |y0| + |y1| of the element's
pair: fp32 adds half a step each for the two products and the sum (3 * 2^-24 h), the sine and cosine (2^-22 h: the reduced turn
is rounded to fp32, half a step of at most pi, and the functions are good to two steps) and, with normalisation, the sum of
squares, the root and two products (at most (D / 8 + 8) 2^-24 h)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from segquant_b200 import ops

DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _check(got, x, pos, axes, theta, pairing, weight, eps=1e-6):
    d = x.shape[-1]
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    want, h, at = y.clone(), y.abs(), 0
    for a, w in enumerate(axes):
        i = torch.arange(w // 2, device=DEV)
        one, two = (at + 2 * i, at + 2 * i + 1) if pairing == "adjacent" else (at + i, at + i + w // 2)
        ang = (pos[..., a, None].double() * theta ** (-2.0 * i.double() / w))[..., None, :]
        c, s = ang.cos(), ang.sin()
        want[..., one], want[..., two] = y[..., one] * c - y[..., two] * s, y[..., one] * s + y[..., two] * c
        h[..., one] = h[..., two] = y[..., one].abs() + y[..., two].abs()
        at += w
    u = torch.finfo(x.dtype).eps / 2
    fp32 = (3 * 2.0 ** -24 + 2.0 ** -22 + (0 if weight is None else (d / 8 + 8) * 2.0 ** -24)) * h
    tol = u * (want.abs() + fp32) + fp32 + (2.0 ** -25 if x.dtype == torch.float16 else 1e-37)       # fp16: half a step of the subnormals
    err = (got.double() - want).abs()
    assert got.dtype == x.dtype and (err <= tol).all(), float((err / tol).max())


CASES = [  # batch, tokens, hq, hk, d, axes, pairing
    (1, 1, 1, 1, 64, (64,), "adjacent"), (1, 1, 32, 8, 128, (128,), "halves"), (2, 333, 24, 24, 64, (16, 24, 24), "adjacent"),
    (1, 700, 5, 1, 128, (44, 42, 42), "adjacent"), (1, 257, 3, 3, 128, (16, 56, 56), "adjacent"), (1, 100, 4, 2, 72, (24, 24, 24), "adjacent"),
    (2, 65, 6, 2, 128, (32, 48, 48), "halves"), (1, 65, 7, 7, 128, (64,), "halves"),                   # columns that are not rotated
    (1, 33, 2, 1, 64, (20, 22, 22), "halves"), (1, 33, 2, 1, 50, (10, 20), "adjacent"), (1, 9, 3, 1, 7, (2, 4), "halves"), (1, 9, 3, 1, 1 + 2, (2,), "adjacent"),
    (1, 40, 2, 2, 256, (64, 96, 96), "halves"), (1, 40, 3, 1, 256, (256,), "adjacent"), (3, 5, 1, 0, 96, (96,), "halves"), (1, 4, 13, 0, 64, (2, 2, 2, 2, 2, 2, 2, 2), "adjacent"),
    (1, 3000, 9, 4, 64, (64,), "adjacent"),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_fp64(native_lib, case, norm, dtype):
    b, t, hq, hk, d, axes, pairing = case
    g = _gen(1)
    q = torch.randn(b, t, hq, d, generator=g, device=DEV).to(dtype)
    k = torch.randn(b, t, hk, d, generator=g, device=DEV).to(dtype) if hk else None
    pos = torch.randint(0, 3000, (b, t, len(axes)), generator=g, device=DEV, dtype=torch.int32)
    w = [(1 + 0.3 * torch.randn(d, generator=g, device=DEV)).to(dtype) if norm else None for _ in range(2)]
    if k is None:
        w[1] = None
    out = ops.rotary(q, k, pos, axes, theta=5e5, pairing=pairing, norm_q=w[0], norm_k=w[1])
    _check(out[0], q, pos, axes, 5e5, pairing, w[0])
    if hk:
        _check(out[1], k, pos, axes, 5e5, pairing, w[1])
    else:
        assert out[1] is None
    # one set of positions for all samples; in place
    out = ops.rotary(q, k, pos[0], axes, theta=100.0, pairing=pairing, norm_q=w[0], norm_k=w[1], eps=1e-3)
    _check(out[0], q, pos[:1], axes, 100.0, pairing, w[0], 1e-3)
    same = q.clone()
    assert ops.rotary(same, k, pos[0], axes, theta=100.0, pairing=pairing, norm_q=w[0], norm_k=w[1], eps=1e-3, out_q=same)[0] is same
    assert torch.equal(same, out[0])
    assert ops.device_status() == 0


@pytest.mark.parametrize("kind", [torch.int32, torch.float32])
def test_far_positions(native_lib, kind):
    """Positions whose angles fp32 could not tell apart, negative ones, and fractions."""
    g = _gen(2)
    pos = torch.tensor([0, 1, -1, 131071, 1000003, 16777213, -16777215, 12345], device=DEV, dtype=kind)[:, None]
    if kind == torch.float32:
        pos = pos + torch.tensor([0.0, 0.5, 0.25, 0.125, 0.0, 0.0, 0.0, 0.75], device=DEV)[:, None]
    for d, pairing in ((64, "adjacent"), (128, "halves"), (50, "halves")):
        q, k = (torch.randn(8, 2, d, generator=g, device=DEV) for _ in range(2))
        out = ops.rotary(q, k, pos, (d,), theta=1e4, pairing=pairing)
        _check(out[0], q, pos, (d,), 1e4, pairing, None)
        _check(out[1], k, pos, (d,), 1e4, pairing, None)


def test_layouts(native_lib):
    g = _gen(3)
    for d, dtype in ((64, torch.bfloat16), (72, torch.float16), (64, torch.float32)):
        buf = torch.randn(2, 70, 3, 4, d, generator=g, device=DEV).to(dtype)
        q, k, _ = buf.unbind(2)
        pos = torch.randint(0, 99, (70, 2), generator=g, device=DEV, dtype=torch.int32)
        call = lambda a, b, **kw: ops.rotary(a, b, pos, (16, 32), **kw)  # noqa: E731
        want = call(q.contiguous(), k.contiguous())
        heads_first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
        odd = torch.empty(q.numel() + 1, dtype=dtype, device=DEV)[1:].view(q.shape).copy_(q)
        for a, b in ((q, k), (heads_first(q), k), (odd, k), (q.transpose(2, 3).contiguous().transpose(2, 3), k)):
            got = call(a, b)
            assert (got[0].double() - want[0].double()).abs().max() <= 2 * torch.finfo(dtype).eps * want[0].abs().max() and torch.equal(got[1], want[1])
        after = buf.clone()
        call(after[:, :, 0], after[:, :, 1], out_q=after[:, :, 0], out_k=after[:, :, 1])     # in place inside the joint buffer
        assert torch.equal(after[:, :, 0], want[0]) and torch.equal(after[:, :, 1], want[1]) and torch.equal(after[:, :, 2], buf[:, :, 2])
        assert torch.equal(call(q, k, out_q=torch.empty_like(q).transpose(1, 2).contiguous().transpose(1, 2))[0], want[0])
        mixed = ops.rotary(q[0], k[0, :, :1].expand(-1, 4, -1), pos, (16, 32))                # packed, one head for all
        assert torch.equal(mixed[0], want[0][0]) and torch.equal(mixed[1][:, 0], want[1][0][:, 0])


def test_streams_and_graphs(native_lib):
    g = _gen(4)
    q, k = (torch.randn(2, 50, 4, 64, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    pos = torch.randint(0, 99, (50, 1), generator=g, device=DEV, dtype=torch.int32)
    want = ops.rotary(q, k, pos, (64,))
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = ops.rotary(q, k, pos, (64,))
    pos += 3
    gr.replay()
    again = ops.rotary(q, k, pos, (64,))
    assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1]) and not torch.equal(out[0], want[0])
    with torch.cuda.stream(torch.cuda.Stream()):
        pos -= 3
        other = ops.rotary(q, k, pos, (64,))
    torch.cuda.synchronize()
    assert torch.equal(other[0], want[0])


def test_nothing_to_do_and_refusals(native_lib):
    q = torch.zeros(2, 8, 4, 64, dtype=torch.bfloat16, device=DEV)
    pos = torch.zeros(8, 1, dtype=torch.int32, device=DEV)
    w = torch.ones(64, dtype=torch.bfloat16, device=DEV)
    assert ops.rotary(q[:0], q[:0], pos, (64,))[0].shape == (0, 8, 4, 64)
    assert ops.rotary(q[:, :0], None, pos[:0], (64,))[0].shape == (2, 0, 4, 64)
    bad = [
        (ValueError, lambda: ops.rotary(q, q, pos, (64,), pairing="both")), (ValueError, lambda: ops.rotary(q, q[:, :4], pos, (64,))),
        (TypeError, lambda: ops.rotary(q, q.half(), pos, (64,))), (ValueError, lambda: ops.rotary(q, q, pos, ())), (ValueError, lambda: ops.rotary(q, q, pos, (2,) * 9)),
        (ValueError, lambda: ops.rotary(q, q, pos[:4], (64,))), (ValueError, lambda: ops.rotary(q, q, pos, (32, 32))), (TypeError, lambda: ops.rotary(q, q, pos.long(), (64,))),
        (TypeError, lambda: ops.rotary(q.double(), q.double(), pos, (64,))), (RuntimeError, lambda: ops.rotary(q, q, pos, (66,))), (RuntimeError, lambda: ops.rotary(q, q, pos, (31,))),
        (ValueError, lambda: ops.rotary(q, q, pos, (64,), norm_q=w)), (ValueError, lambda: ops.rotary(q, None, pos, (64,), norm_k=w)),
        (ValueError, lambda: ops.rotary(q, q, pos, (64,), norm_q=w[:32], norm_k=w)), (ValueError, lambda: ops.rotary(q, q, pos, (64,), out_q=q[:1])),
        (ValueError, lambda: ops.rotary(q, None, pos, (64,), out_k=q)), (RuntimeError, lambda: ops.rotary(q, q, pos, (64,), theta=0.0)),
        (RuntimeError, lambda: ops.rotary(q.cpu(), None, pos, (64,))), (RuntimeError, lambda: ops.rotary(q.float().requires_grad_(), None, pos, (64,))),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("hq,hk,d,axes,pairing", [(9, 17, 33, (6, 10), "halves"), (5, 3, 100, (20, 22, 22), "halves"), (11, 2, 251, (80, 90, 80), "adjacent"),
                                                 (7, 9, 129, (128,), "halves")])
def test_odd_layouts_in_place(native_lib, hq, hk, d, axes, pairing, norm, dtype):
    """Views that start at an odd element, heads that no step of several divides, written in place; what lies between them stays."""
    g = _gen(11)
    buf = torch.randn(2, 37, hq + hk, d + 3, generator=g, device=DEV).to(dtype)
    before = buf.clone()
    cut = lambda t: (t[:, :, :hq, 1:d + 1], t[:, :, hq:, 1:d + 1])  # noqa: E731
    q, k = cut(buf)
    pos = torch.randint(0, 500, (37, len(axes)), generator=g, device=DEV, dtype=torch.int32)
    w = [torch.randn(d, generator=g, device=DEV).to(dtype) for _ in range(2)] if norm else [None, None]
    ops.rotary(q, k, pos, axes, pairing=pairing, norm_q=w[0], norm_k=w[1], out_q=q, out_k=k)
    for got, x, weight in zip(cut(buf), cut(before), w):
        _check(got, x, pos[None], axes, 10000.0, pairing, weight)
    assert torch.equal(buf[..., 0], before[..., 0]) and torch.equal(buf[..., d + 1:], before[..., d + 1:])


def test_columns_behind_the_axes_are_not_mixed(native_lib):
    x = torch.randn(1, 6, 3, 51, generator=_gen(12), device=DEV)
    bad = x.clone()
    bad[..., 41], bad[..., 50] = float("nan"), float("inf")
    pos = torch.arange(6, device=DEV, dtype=torch.int32)[:, None]
    out = lambda t: ops.rotary(t, t, pos, (40,))[0]  # noqa: E731
    clean, got = out(x), out(bad)
    keep = torch.ones(51, dtype=torch.bool, device=DEV)
    keep[41] = keep[50] = False
    assert torch.equal(clean[..., keep], got[..., keep]) and torch.isnan(got[..., 41]).all() and torch.isinf(got[..., 50]).all()
    assert torch.equal(clean[..., 40:], x[..., 40:])
