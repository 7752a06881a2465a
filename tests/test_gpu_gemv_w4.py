"""GPU: int4 layers with up to 8 rows run on the weight-streaming kernel.  Its results have to be the bits of the tensor-core
path (the integer sums of a unit are exact, the fp32 steps and their order are the same) and agree with fp64: per output
U units, each rounded twice for its reciprocal scale(s) and once for the running sum, so (U + 4) 2^-23 sum |terms| and one
rounding to the output type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from segquant_b200 import _lib as L
from segquant_b200 import ops

DEV = "cuda"


def _case(m, n, k, bounds, group, per_token, dual, dtype, bias, sw_dtype=torch.float32, column_major=False, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randint(-128, 128, (1, m, k), generator=g, device=DEV, dtype=torch.int8)
    xq, xn = (x.clamp(min=0), x.clamp(max=0)) if dual else (x, None)
    wq = torch.randint(0, 256, (1, n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    S = len(bounds) - 1
    sx = torch.rand(S * (m if per_token else 1), generator=g, device=DEV) * 20 + 20
    sxn = sx * 3 if dual else None
    groups = -(-k // group) if group else 1          # the last group may be a part of one
    sw = (torch.rand(groups, n, generator=g, device=DEV) * 50 + 50).to(sw_dtype)
    strides, sw_arg = ((0, 0, 1, groups), sw.t().contiguous()) if column_major else ((0, 0, n, 1), sw)
    b = torch.randn(n, generator=g, device=DEV).to(torch.float32 if dtype == torch.float32 else dtype) if bias else None

    def run(**kw):
        return ops.gemm(L.SQ_GEMM_W4A8, xq.view(torch.uint8), wq, n, bounds, sx, sw_arg, xq_neg=None if xn is None else xn.view(torch.uint8), sx_neg=sxn,
                        per_token=per_token, group_size=group, sw_strides=strides, bias=b, out_dtype=dtype, **kw)

    def exact():
        byte = wq[0].long()
        w = torch.stack([((byte & 15) ^ 8) - 8, ((byte >> 4) ^ 8) - 8], dim=-1).view(n, k).double()
        y, a, units = torch.zeros(m, n, dtype=torch.float64, device=DEV), torch.zeros(m, n, dtype=torch.float64, device=DEV), 0
        cuts = sorted(set(bounds) | set(range(0, k, group) if group else ()) | {k})
        for k0, k1 in zip(cuts, cuts[1:]):
            s = max(i for i in range(S) if bounds[i] <= k0)
            units += 1
            for c, scale in ((xq, sx), (xn, sxn)):
                if c is None:
                    continue
                sc = scale.view(S, -1)[s].double()[:, None]
                t = c[0, :, k0:k1].double() @ w[:, k0:k1].T / (sc * sw[k0 // group if group else 0].double()[None])
                y, a = y + t, a + t.abs()
        if b is not None:
            y, a = y + b.double(), a + b.double().abs()
        return y, a * (2 * units + 4) * 2.0 ** -23 + y.abs() * torch.finfo(dtype).eps / 2 + 1e-30
    return run, exact


CASES = [  # m, n, k, bounds, group, per token, dual, dtype, bias
    (1, 1, 32, [0, 32], 0, False, False, torch.float32, False), (1, 520, 512, [0, 512], 64, True, False, torch.float32, True),
    (2, 9216, 1536, [0, 1536], 128, False, True, torch.bfloat16, True), (4, 1000, 12288, [0, 12288], 128, True, False, torch.float16, True),
    (3, 77, 3200, [0, 1024, 3200], 128, False, False, torch.float32, False), (4, 41, 2048, [0, 96, 2048], 32, True, True, torch.bfloat16, True),
    (3, 64, 8192, [0, 8192], 0, False, False, torch.float32, False), (8, 1000, 12288, [0, 12288], 128, True, False, torch.float16, True),
    (5, 70, 1536, [0, 512, 1536], 128, False, True, torch.bfloat16, True), (7, 3000, 6144, [0, 6144], 64, True, True, torch.float32, True),
    (6, 20000, 1024, [0, 1024], 0, True, False, torch.float32, False), (4, 50, 12288, [0, 12288], 32, True, True, torch.float32, True),
    (2, 33, 1248, [0, 192, 384, 1248], 96, True, False, torch.bfloat16, True), (8, 17, 160, [0, 32, 64, 160], 0, False, True, torch.float32, True),
    (1, 4099, 384, [0, 384], 256, False, False, torch.bfloat16, False), (8, 16, 65536, [0, 65536], 0, True, False, torch.float32, False),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_same_bits_as_the_tensor_core_path(native_lib, case):
    run, exact = _case(*case)
    got = run()
    ops.set_gemm_schedule(no_gemv=1)
    try:
        tiles = run()
    finally:
        ops.set_gemm_schedule()
    assert torch.equal(got, tiles)
    want, tol = exact()
    assert ((got[0].double() - want).abs() <= tol).all()
    assert ops.device_status() == 0


@pytest.mark.parametrize("sw_dtype,column_major", [(torch.bfloat16, False), (torch.float32, True), (torch.bfloat16, True)])
def test_scale_layouts(native_lib, sw_dtype, column_major):
    run, exact = _case(3, 300, 1024, [0, 1024], 128, False, False, torch.float32, True, sw_dtype, column_major)
    want, tol = exact()
    assert ((run()[0].double() - want).abs() <= tol).all()


def test_strided_output_and_graph(native_lib):
    run, _ = _case(4, 200, 512, [0, 512], 64, True, False, torch.bfloat16, True)
    want = run()
    wide = torch.full((1, 4, 456), 3.0, dtype=torch.bfloat16, device=DEV)
    run(out=wide[:, :, 128:328], y_strides=(4 * 456, 456))
    assert torch.equal(wide[:, :, 128:328], want) and (wide[:, :, :128] == 3.0).all() and (wide[:, :, 328:] == 3.0).all()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = run()
    out.zero_()
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_layer_forward_with_few_rows(native_lib):
    """A SegmentLinear with int4 weights and group scales gives a row the same bits alone as among many."""
    from segquant_b200.layers.SegmentLinear import SegmentLinear
    g = torch.Generator().manual_seed(3)
    w, b, x = torch.randn(384, 512, generator=g) * 0.05, torch.randn(384, generator=g), torch.randn(64, 512, generator=g)
    lin = SegmentLinear(512, 384, bias=True, seg_mode="input", chunks=2, custom_weight_tensor=w.to(DEV), custom_bias_tensor=b.to(DEV), input_quant_type="int8",
                        weight_quant_type="int4", input_quant_args={"real_quant": True, "axis": None}, weight_quant_args={"real_quant": True, "axis": 1}, device=DEV)
    xd = x.to(torch.bfloat16).to(DEV)
    lin.calibrate(xd)
    lin.finish_calibrate()
    whole = lin(xd)
    for m in (1, 2, 4, 7, 8):
        assert torch.equal(lin(xd[:m]), whole[:m])
