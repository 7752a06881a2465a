"""GPU: the denoise step with this library's attention, rotary positions and 4-bit modulation weights, together, as a model uses
them: eagerly, over two streams, captured into a graph and replayed.

The attention's inputs are the same bf16 tensors on both sides of each comparison up to the first block's attention, which both
compute to bf16; from there on the two differ by bf16 roundings that the quantised layers pass on as single steps of int8, as
they do between the fused and the unfused step (cos > 0.999 there and here)."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

from segquant_b200 import ops
from segquant_b200.mmdit import GraphedStep, JointBlock, SyntheticMMDiT, grid_positions, synthetic_inputs

DEV = "cuda"
SMALL = dict(blocks=3, hidden=512, heads=8, img_tokens=144, txt_tokens=37)


def _inputs(batch=2, seed=1):
    return synthetic_inputs(batch, DEV, img_tokens=144, txt_tokens=37, hidden=512, seed=seed)


def _cos(a, b):
    return float(F.cosine_similarity(a.double().flatten(), b.double().flatten(), dim=0))


def test_fused_attention_step_against_torch(native_lib):
    ins = _inputs()
    ref, fused = (SyntheticMMDiT(DEV, **SMALL, attention=a) for a in ("torch", "fused"))
    ref.calibrate(*ins)
    fused.calibrate(*ins)
    assert _cos(fused(*ins), ref(*ins)) > 0.999


def test_rotary_norm_and_int4_modulation_step(native_lib):
    ins = _inputs()
    kw = dict(rotary_axes=(16, 24, 24), qk_norm=True, modulation_weights="int4")
    ref, model = (SyntheticMMDiT(DEV, **SMALL, attention=a, **kw) for a in ("torch", "fused"))
    ref.calibrate(*ins)
    model.calibrate(*ins)
    want = model(*ins)
    assert _cos(want, ref(*ins)) > 0.999
    model.two_streams = False
    assert torch.equal(model(*ins), want)
    # the skinny int4 kernel serves the modulations (2 rows) with the bits of the tensor-core path
    ops.set_gemm_schedule(no_gemv=1)
    try:
        assert torch.equal(model(*ins), want)
    finally:
        ops.set_gemm_schedule()
    model.two_streams = True
    step = GraphedStep(model, *ins)
    assert step.launches_per_replay > 0
    other = _inputs(seed=2)
    eager = model(*other).clone()
    assert torch.equal(step(*other), eager) and torch.equal(step(*ins), want)
    assert ops.device_status() == 0


def test_rotary_in_the_joint_buffer(native_lib):
    """The block turns q and k in place and leaves v: against a plain restatement of the same attention."""
    gen = torch.Generator().manual_seed(3)
    blk = JointBlock(512, 8, gen, DEV, torch.bfloat16, last=True, out_proj_segments=1, attention="fused", rotary_axes=(16, 24, 24), qk_norm=True)
    g = torch.Generator(device=DEV).manual_seed(4)
    img, txt = (torch.randn(2, n, 512, generator=g, device=DEV).to(torch.bfloat16) for n in (144, 37))
    c = torch.randn(2, 512, generator=g, device=DEV).to(torch.bfloat16)
    seen = {}

    def call(layer, x, out=None, pre_act=None):
        if layer is blk.to_out:
            seen["a_img"] = x.clone()
        y = F.linear(x if pre_act is None else F.gelu(x, approximate="tanh"), layer.w, layer.b)
        return y if out is None else out.copy_(y)

    def norm_call(layers, x, shift, scale, outs=None, residual=None):
        ys = [call(lay, x, o) for lay, o in zip(layers, outs or [None] * len(layers))]
        return ys, x

    with pytest.raises(RuntimeError, match="positions"):
        blk.forward(img, txt, c, call, norm_call)
    blk.positions = grid_positions(144, 37, DEV)
    blk.forward(img, txt, c, call, norm_call)
    proj = lambda a, b: torch.cat([F.linear(img, a.w, a.b), F.linear(txt, b.w, b.b)], dim=1).view(2, 181, 8, 64).double()  # noqa: E731
    q, k, v = proj(blk.to_q, blk.add_q), proj(blk.to_k, blk.add_k), proj(blk.to_v, blk.add_v)
    cols = [blk.positions[:, a].double()[:, None] * 10000.0 ** (-torch.arange(0, w, 2, device=DEV).double() / w) for a, w in enumerate((16, 24, 24))]
    ang = torch.cat(cols, dim=1)[:, None]
    turn = lambda x: torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:-1], 32, 2).contiguous()) * torch.polar(torch.ones_like(ang), ang)).flatten(-2)  # noqa: E731
    rms = lambda x: x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    q, k = turn(rms(q)).transpose(1, 2), turn(rms(k)).transpose(1, 2)
    want = (torch.softmax(q @ k.transpose(2, 3) / 8.0, dim=-1) @ v.transpose(1, 2)).transpose(1, 2).reshape(2, 181, 512)[:, :144]
    # q and k are rounded to bf16 once more than here (2^-8 each of unit-size heads: scores move by at most 2 * 2^-8 * 8), p and
    # the result once each
    err = (seen["a_img"].double() - want).abs().max()
    assert err <= want.abs().max() * (2 * 2.0 ** -8) + v.abs().max() * 2 * (2 * 2.0 ** -8 * 8), float(err)


def test_refused_options(native_lib):
    with pytest.raises(ValueError):
        SyntheticMMDiT(DEV, **SMALL, attention="other")
    with pytest.raises(ValueError):
        SyntheticMMDiT(DEV, **SMALL, qk_norm=True)
    with pytest.raises(ValueError):
        grid_positions(150, 3, DEV)
