"""GPU: what a joint block does between its projections and its output projection, element by element against fp64.

The projections are taken from the block's own calls, so that the comparison starts from the same bf16 values:
  * q and k behind the heads' normalisation and the rotation: one rounding (u = eps / 2, half a step relative to the value) and
    fp32 terms, 3 * 2^-24 + 2^-22 of |y0| + |y1| of a pair for the rotation and (D / 8 + 8) 2^-24 for the normalisation; v: the same bits;
  * the attention of those q, k, v: A (u + 2 eta + n 2^-23) + u |o| with A = sum p |v|, eta = (D + 1.5) 2^-23 sum |q k| scale + 4e-6.
References without the normalisation, without the rotation, with positions of one axis left out, or with equal weights violate the
bounds: they are tight enough to tell."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

from segquant_b200 import ops
from segquant_b200.mmdit import JointBlock, grid_positions

DEV = "cuda"
HEADS, D, TI, TT = 8, 64, 144, 37
AXES = (16, 24, 24)
U = torch.finfo(torch.bfloat16).eps / 2


def _norm(x):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)


def _turn(x, pos):
    """(value, |y0| + |y1| of the pair) of the rotation in fp64; pos (tokens, 3)."""
    ang = torch.cat([pos[:, a].double()[:, None] * 10000.0 ** (-torch.arange(0, w, 2, device=x.device).double() / w) for a, w in enumerate(AXES)], dim=1)[:, None]
    y0, y1 = x[..., 0::2], x[..., 1::2]
    h = y0.abs() + y1.abs()
    out = torch.stack([y0 * ang.cos() - y1 * ang.sin(), y0 * ang.sin() + y1 * ang.cos()], dim=-1).flatten(-2)
    return out, torch.stack([h, h], dim=-1).flatten(-2)


def _inside(got, want, tol):
    return bool(((got.double() - want).abs() <= tol).all())


def _q_inside(got, x, pos, weight, norm=True, turn=True):
    y = _norm(x.double()) * weight.double() if norm else x.double()
    want, h = _turn(y, pos) if turn else (y, y.abs())
    fp32 = (3 * 2.0 ** -24 + 2.0 ** -22 + (D / 8 + 8) * 2.0 ** -24) * h
    return _inside(got, want, U * (want.abs() + fp32) + fp32 + 1e-37)


def _out_inside(got, q, k, v, uniform=False):
    q, k, v = (t.double().transpose(1, 2) for t in (q, k, v))
    n = k.shape[2]
    p = torch.softmax(q @ k.transpose(2, 3) * D ** -0.5 * (0.0 if uniform else 1.0), dim=-1)
    eta = (D + 1.5) * 2.0 ** -23 * (q.abs() @ k.abs().transpose(2, 3)).amax(-1, keepdim=True) * D ** -0.5 + 4e-6
    o, a = p @ v, p @ v.abs()
    return _inside(got.transpose(1, 2), o, a * (U + 2 * eta + n * 2.0 ** -23) + U * o.abs())


def _run(monkeypatch, rotary_axes, qk_norm):
    gen = torch.Generator().manual_seed(3)
    blk = JointBlock(HEADS * D, HEADS, gen, DEV, torch.bfloat16, last=False, out_proj_segments=1, attention="fused", rotary_axes=rotary_axes, qk_norm=qk_norm)
    if rotary_axes:
        blk.positions = grid_positions(TI, TT, DEV)
    if qk_norm:                                                  # weights of their own, so that q's cannot stand in for k's
        g = torch.Generator(device=DEV).manual_seed(6)
        blk.norm_q, blk.norm_k = ((1.0 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(torch.bfloat16) for _ in range(2))
    g = torch.Generator(device=DEV).manual_seed(4)
    img, txt = (4.0 * torch.randn(2, n, HEADS * D, generator=g, device=DEV).to(torch.bfloat16) for n in (TI, TT))
    c = torch.randn(2, HEADS * D, generator=g, device=DEV).to(torch.bfloat16)
    seen, passed = {}, {}

    def call(layer, x, out=None, pre_act=None):
        y = F.linear(x if pre_act is None else F.gelu(x, approximate="tanh"), layer.w, layer.b)
        seen[layer] = (x.clone(), y.clone())
        return y if out is None else out.copy_(y)

    def norm_call(layers, x, shift, scale, outs=None, residual=None):
        return [call(lay, x, o) for lay, o in zip(layers, outs or [None] * len(layers))], x

    real = ops.attention

    def spy(q, k, v, **kw):
        passed.update(q=q.clone(), k=k.clone(), v=v.clone())
        return real(q, k, v, **kw)

    monkeypatch.setattr(ops, "attention", spy)
    blk.forward(img, txt, c, call, norm_call)
    proj = {n: torch.cat([seen[a][1], seen[b][1]], dim=1).view(2, TI + TT, HEADS, D)
            for n, a, b in (("q", blk.to_q, blk.add_q), ("k", blk.to_k, blk.add_k), ("v", blk.to_v, blk.add_v))}
    out = torch.cat([seen[blk.to_out][0], seen[blk.to_add_out][0]], dim=1).view(2, TI + TT, HEADS, D)
    return blk, proj, passed, out


def test_normalised_and_turned(native_lib, monkeypatch):
    blk, proj, passed, out = _run(monkeypatch, AXES, True)
    pos = blk.positions
    for n, w, other in (("q", blk.norm_q, blk.norm_k), ("k", blk.norm_k, blk.norm_q)):
        assert _q_inside(passed[n], proj[n], pos, w)
        assert not _q_inside(passed[n], proj[n], pos, w, norm=False) and not _q_inside(passed[n], proj[n], pos, w, turn=False)
        assert not _q_inside(passed[n], proj[n], pos, other)
        for a in range(3):
            part = pos.clone()
            part[:, a] = 0
            assert not _q_inside(passed[n], proj[n], part, w)
    assert torch.equal(passed["v"], proj["v"])
    assert _out_inside(out, passed["q"], passed["k"], passed["v"])
    assert not _out_inside(out, passed["q"], passed["k"], passed["v"], uniform=True)
    assert not _out_inside(out, proj["q"], proj["k"], proj["v"]) and not _out_inside(out, passed["q"], proj["k"], passed["v"])
    assert ops.device_status() == 0


def test_without_rotary(native_lib, monkeypatch):
    blk, proj, passed, out = _run(monkeypatch, None, False)
    for n in ("q", "k", "v"):
        assert torch.equal(passed[n], proj[n])
    assert _out_inside(out, proj["q"], proj["k"], proj["v"]) and not _out_inside(out, proj["q"], proj["k"], proj["v"], uniform=True)
