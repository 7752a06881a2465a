"""torch-tensor front end of the C ABI (include/segquant_b200.h).

torch is used here only for device memory and the current stream; all arithmetic happens in the
sm_100a kernels of libsegquant_b200.so.  There is no CPU implementation: every function raises if
its tensors are not on a CUDA device.

The two functions at the bottom keep the tensor contract of the reference's pybind functions
(segquant/src/real_quant/seg_utils.h:122-161, real_gemm.cu:643-894); `seg_linear` is the fused
layer forward that SegmentLinear uses.
"""
import ctypes
import functools
import struct

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _lib as L

_DT = {torch.float32: L.SQ_F32, torch.float16: L.SQ_F16, torch.bfloat16: L.SQ_BF16}

# kernel_type string (f"W{weight}A{input}", segquant/layers/SegmentLinear.py:103)
#   -> (GEMM kind, activation storage, weight storage)
KERNELS = {
    "Wint8Aint8": (L.SQ_GEMM_W8A8_I8, L.SQ_Q_INT8, L.SQ_Q_INT8),
    "Wfpe4m3Afpe4m3": (L.SQ_GEMM_W8A8_F8, L.SQ_Q_E4M3, L.SQ_Q_E4M3),
    "Wint4Aint8": (L.SQ_GEMM_W4A8, L.SQ_Q_INT8, L.SQ_Q_INT4),
}

launch_count = 0  # kernels of this library launched by this process (bench.py reports it)


def _stream(t):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


# Argument blocks of the operators that are short enough for their Python call to count, packed in one go (setting the fields of
# a ctypes.Structure one by one takes three times as long); the layouts are those of _lib's structures.
_GEMM = struct.Struct("@ii4qPPqqPqqii%dsiiPPqqqPqqqqPiiqPqqPii%dPqq" % (4 * (L.SQ_MAX_SEGS + 1), L.SQ_MAX_PEERS))
_ATTENTION = struct.Struct("@5Pii3qiiii12q4PfiPq")
_ROTARY = struct.Struct("@4Piiqqiiii%ds12qPqqifdPP" % (4 * L.SQ_ROTARY_MAX_AXES))
assert (_GEMM.size, _ATTENTION.size, _ROTARY.size) == tuple(ctypes.sizeof(c) for c in (L.GemmArgs, L.AttentionArgs, L.RotaryArgs))
_NO_PEERS = (0,) * L.SQ_MAX_PEERS
_raw_stream = torch._C._cuda_getCurrentRawStream


def _run(fn, what, dev, *args):
    """Calls a C entry point with the current stream of device `dev` (made current for the call if it is not) and checks its
    status.  Without a context manager where it can be: a small operator is done before its Python call returns."""
    if torch.cuda.current_device() == dev:
        status = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, _raw_stream(dev))
    if status < 0:
        L.check(status, what)


def _need_cuda(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError("segquant_b200: tensors must live on a CUDA device (there is no CPU path)")


def _dt(t):
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError(f"segquant_b200: unsupported floating dtype {t.dtype}") from None


def _f32(t, device):
    if not isinstance(t, torch.Tensor):
        t = torch.tensor(t, dtype=torch.float32, device=device)
    return t.to(device=device, dtype=torch.float32).contiguous()


def uniform_bounds(K, segments):
    if K % segments:
        raise ValueError(f"K={K} is not divisible into {segments} equal segments")
    step = K // segments
    return [i * step for i in range(segments + 1)]


# ---------------------------------------------------------------------------------------------
# activation quantise
# ---------------------------------------------------------------------------------------------
PRE_ACTS = {None: L.SQ_ACT_NONE, "gelu_tanh": L.SQ_ACT_GELU_TANH, "silu": L.SQ_ACT_SILU}


def quantize_act(x, bounds, sx, sx_neg=None, out_kind=L.SQ_Q_INT8, per_token=False, smooth=None,
                 out=None, out_neg=None, shared_scales=False, pre_act=None):
    """x: (B, M, K) view (any batch / row stride, K contiguous) or (M, K).

    sx: (B*S,) or (B*S*M,) float32 in (batch, segment[, row]) order, or (S,) used by every batch
    when shared_scales is set.  Returns (xq, xq_neg) uint8 tensors of shape (B, M, K) (contiguous).
    `bounds` cuts K into the S segments.  pre_act ("gelu_tanh" / "silu") applies that activation to x, in fp32,
    inside the kernel, so the activation in front of a layer costs no pass over memory of its own."""
    global launch_count
    _need_cuda(x, sx, sx_neg)
    if pre_act not in PRE_ACTS:
        raise ValueError(f"pre_act must be one of {list(PRE_ACTS)}")
    if x.dim() == 2:
        x = x.unsqueeze(0)
    if x.stride(-1) != 1:
        x = x.contiguous()
    B, M, K = x.shape
    S = len(bounds) - 1
    dual = sx_neg is not None
    xq = out if out is not None else torch.empty((B, M, K), dtype=torch.uint8, device=x.device)
    xqn = (out_neg if out_neg is not None else torch.empty((B, M, K), dtype=torch.uint8, device=x.device)) if dual else None
    if x.numel() == 0:
        return xq, xqn
    a = L.ActQuantArgs()
    a.x_dev = x.data_ptr()
    a.x_dtype = _dt(x)
    a.out_kind = out_kind
    a.batch, a.M, a.K = B, M, K
    a.x_batch_stride, a.x_row_stride = (x.stride(0) if B > 1 else 0), x.stride(1)
    a.num_segs = S
    L.set_bounds(a.seg_bounds, bounds)
    a.sx_dev = sx.data_ptr()
    a.sx_neg_dev = sx_neg.data_ptr() if dual else None
    if per_token:
        a.sx_batch_stride, a.sx_seg_stride, a.sx_row_stride = S * M, M, 1
    else:
        a.sx_batch_stride, a.sx_seg_stride, a.sx_row_stride = S, 1, 0
    if shared_scales:
        a.sx_batch_stride = 0
    a.smooth_dev = smooth.data_ptr() if smooth is not None else None
    a.pre_act = PRE_ACTS[pre_act]
    a.xq_dev = xq.data_ptr()
    a.xq_neg_dev = xqn.data_ptr() if dual else None
    a.xq_batch_stride, a.xq_row_stride = M * K, K
    with torch.cuda.device(x.device):
        L.check(L.load().sq_quantize_act(ctypes.byref(a), _stream(x)), "sq_quantize_act")
    launch_count += 1
    return xq, xqn


def norm_quantize_act(x, bounds, sx, sx_neg=None, out_kind=L.SQ_Q_INT8, shift=None, scale=None, eps=1e-6, residual=None):
    """LayerNorm(x) * (1 + scale) + shift, quantised with the static per-segment scales, in one pass over x.

    x: (B, T, K) with contiguous rows; shift / scale: (B, K) in x's dtype (or both None for a plain LayerNorm);
    sx (and sx_neg for DualScale): (S,) float32 shared by all batches.  Returns (xq, xq_neg) uint8 (B, T, K).

    residual=(gate (B, K), y (B, T, K)): the stream is first updated, x' = x + gate * y (bit-identical to torch.addcmul),
    in the same pass; returns (xq, xq_neg, x') with x' a new tensor of x's dtype."""
    global launch_count
    _need_cuda(x, sx, sx_neg, shift, scale)
    if x.dim() != 3 or x.stride(-1) != 1:
        raise ValueError("norm_quantize_act needs a (B, T, K) tensor with contiguous rows")
    B, M, K = x.shape
    dual = sx_neg is not None
    xq = torch.empty((B, M, K), dtype=torch.uint8, device=x.device)
    xqn = torch.empty((B, M, K), dtype=torch.uint8, device=x.device) if dual else None
    if x.numel() == 0:
        return (xq, xqn) if residual is None else (xq, xqn, x.clone())
    a = L.ActQuantArgs()
    a.x_dev, a.x_dtype, a.out_kind = x.data_ptr(), _dt(x), out_kind
    a.batch, a.M, a.K = B, M, K
    a.x_batch_stride, a.x_row_stride = (x.stride(0) if B > 1 else 0), x.stride(1)
    a.num_segs = len(bounds) - 1
    L.set_bounds(a.seg_bounds, bounds)
    a.sx_dev = sx.data_ptr()
    a.sx_neg_dev = sx_neg.data_ptr() if dual else None
    a.sx_batch_stride, a.sx_seg_stride, a.sx_row_stride = 0, 1, 0
    a.xq_dev = xq.data_ptr()
    a.xq_neg_dev = xqn.data_ptr() if dual else None
    a.xq_batch_stride, a.xq_row_stride = M * K, K
    mod_bs = 0
    if shift is not None:
        if shift.dtype != x.dtype or scale.dtype != x.dtype or shift.shape != (B, K) or scale.shape != (B, K):
            raise ValueError("shift / scale must be (B, K) tensors of x's dtype")
        if shift.stride(-1) != 1 or scale.stride(-1) != 1 or (B > 1 and shift.stride(0) != scale.stride(0)):
            shift, scale = shift.contiguous(), scale.contiguous()     # views with one common row stride are read in place
        mod_bs = shift.stride(0) if B > 1 else 0
    res, x_new = None, None
    if residual is not None:
        gate, y = residual
        _need_cuda(gate, y)
        if y.shape != x.shape or y.dtype != x.dtype or y.stride(-1) != 1 or gate.shape != (B, K) or gate.dtype != x.dtype:
            raise ValueError("residual=(gate (B, K), y (B, T, K)) in x's dtype, rows contiguous")
        if gate.stride(-1) != 1:
            gate = gate.contiguous()
        x_new = torch.empty((B, M, K), dtype=x.dtype, device=x.device)
        res = L.NormResidual()
        res.y_dev, res.gate_dev, res.x_out_dev = y.data_ptr(), gate.data_ptr(), x_new.data_ptr()
        res.y_batch_stride, res.y_row_stride = (y.stride(0) if B > 1 else 0), y.stride(1)
        res.gate_batch_stride = gate.stride(0) if B > 1 else 0
        res.x_out_batch_stride, res.x_out_row_stride = M * K, K
    with torch.cuda.device(x.device):
        L.check(L.load().sq_residual_norm_quantize_act(ctypes.byref(a), shift.data_ptr() if shift is not None else None,
                                                       scale.data_ptr() if scale is not None else None, mod_bs, float(eps),
                                                       ctypes.byref(res) if res is not None else None, _stream(x)),
                "sq_norm_quantize_act")
    launch_count += 1
    return (xq, xqn) if residual is None else (xq, xqn, x_new)


def gated_residual(x, gate, y, out=None):
    """x + gate.unsqueeze(1) * y for 16-bit (B, T, K) tensors x, y (contiguous rows) and a (B, K) gate, bit-identical to
    torch.addcmul; `out` may be x itself."""
    global launch_count
    _need_cuda(x, gate, y)
    if x.dim() != 3 or y.shape != x.shape or gate.shape != (x.shape[0], x.shape[2]) or x.stride(-1) != 1 or y.stride(-1) != 1:
        raise ValueError("gated_residual needs (B, T, K) tensors x, y with contiguous rows and a (B, K) gate")
    if not (x.dtype == y.dtype == gate.dtype) or x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("gated_residual: x, gate and y must share a 16-bit dtype")
    if gate.stride(-1) != 1:
        gate = gate.contiguous()
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device) if out is None else out
    if x.numel() == 0:
        return out
    B, M, K = x.shape
    a = L.GatedResidualArgs()
    a.x_dev, a.gate_dev, a.y_dev, a.out_dev = x.data_ptr(), gate.data_ptr(), y.data_ptr(), out.data_ptr()
    a.dtype = _dt(x)
    a.batch, a.M, a.K = B, M, K
    a.x_batch_stride, a.x_row_stride = (x.stride(0) if B > 1 else 0), x.stride(1)
    a.y_batch_stride, a.y_row_stride = (y.stride(0) if B > 1 else 0), y.stride(1)
    a.out_batch_stride, a.out_row_stride = (out.stride(0) if B > 1 else 0), out.stride(1)
    a.gate_batch_stride = gate.stride(0) if B > 1 else 0
    with torch.cuda.device(x.device):
        L.check(L.load().sq_gated_residual(ctypes.byref(a), _stream(x)), "sq_gated_residual")
    launch_count += 1
    return out


def quantize_act_dynamic(x, bounds, out_kind=L.SQ_Q_INT8, dual=False, smooth=None):
    """Per-token dynamic scales + quantise in one launch.  x (M, K).  Returns
    (xq, xq_neg, sx, sx_neg) with scales of shape (S, M).  smooth: (K,) float32 divisors, already rounded
    to x's dtype; the kernel calibrates and quantises round_dtype(x / smooth)."""
    global launch_count
    _need_cuda(x, smooth)
    if x.dim() != 2 or x.stride(-1) != 1:
        x = x.reshape(-1, x.shape[-1]).contiguous()
    M, K = x.shape
    S = len(bounds) - 1
    xq = torch.empty((M, K), dtype=torch.uint8, device=x.device)
    xqn = torch.empty((M, K), dtype=torch.uint8, device=x.device) if dual else None
    sx = torch.empty((S, M), dtype=torch.float32, device=x.device)
    sxn = torch.empty((S, M), dtype=torch.float32, device=x.device) if dual else None
    a = L.ActQuantArgs()
    a.x_dev = x.data_ptr()
    a.x_dtype = _dt(x)
    a.out_kind = out_kind
    a.batch, a.M, a.K = 1, M, K
    a.x_batch_stride, a.x_row_stride = 0, x.stride(0)
    a.num_segs = S
    L.set_bounds(a.seg_bounds, bounds)
    a.xq_dev = xq.data_ptr()
    a.xq_neg_dev = xqn.data_ptr() if dual else None
    a.xq_batch_stride, a.xq_row_stride = M * K, K
    a.smooth_dev = smooth.data_ptr() if smooth is not None else None
    with torch.cuda.device(x.device):
        L.check(L.load().sq_quantize_act_dynamic(ctypes.byref(a), ctypes.c_void_p(sx.data_ptr()),
                                                 ctypes.c_void_p(sxn.data_ptr()) if dual else None, _stream(x)),
                "sq_quantize_act_dynamic")
    launch_count += 1
    return xq, xqn, sx, sxn


# ---------------------------------------------------------------------------------------------
# outputs that are given
# ---------------------------------------------------------------------------------------------
def _meets(r, width, dims, moved):
    """Whether r + sum d_i stride_i lies within (-width, width) for some d; dims: (stride, least d, greatest d) from the largest
    stride on.  Exact: d is tried as far as the smaller strides can make up for it, once or twice a dimension in a nested layout.
    moved false: d = 0 does not count."""
    if not dims:
        return moved and -width < r < width
    (s, lo, hi), rest = dims[0], dims[1:]
    least, most = sum(t * l for t, l, _ in rest), sum(t * h for t, _, h in rest)
    first, last = max(lo, (-width - most - r) // s + 1), min(hi, -((r + least - width) // s) - 1)
    return any(_meets(r + d * s, width, rest, moved or d != 0) for d in range(first, last + 1))


@functools.lru_cache(maxsize=1024)
def _layout_overlaps_itself(shape, stride):
    dims = [(s, 1 - n, n - 1) for n, s in zip(shape[:-1], stride) if n > 1]
    return any(s == 0 for s, _, _ in dims) or _meets(0, shape[-1], sorted(dims, reverse=True), False)


def _overlaps_itself(t):
    return not t.is_contiguous() and t.numel() > 0 and _layout_overlaps_itself(t.shape, t.stride())


@functools.lru_cache(maxsize=1024)
def _layouts_overlap(gap, es, shape_a, stride_a, shape_b, stride_b):
    reach = lambda shape, stride: es * (sum((n - 1) * s for n, s in zip(shape, stride)) + 1)  # noqa: E731
    if gap >= reach(shape_b, stride_b) or -gap >= reach(shape_a, stride_a):
        return False
    dims = []
    for na, sa, nb, sb in zip(shape_a[:-1], stride_a, shape_b[:-1], stride_b):
        if na == 1 and nb == 1:
            continue
        if na > 1 and nb > 1 and sa != sb:
            return False
        s = sa if na > 1 else sb
        if s:
            dims.append((es * s, 1 - nb, na - 1))
    return _meets(gap, es * shape_a[-1], sorted(dims, reverse=True), True)


def _overlap(a, b):
    """Whether a and b (one dtype, last dimensions contiguous and as wide) share an element: exactly where their strides are the same, else
    where they start at the same address or lie apart as a whole.  A matter of the layouts and the distance between the two, which
    a program's calls repeat: worked out once for each (13 us in a buffer of q | k | v)."""
    if not a.numel() or not b.numel():
        return False
    gap = a.data_ptr() - b.data_ptr()
    return gap == 0 or (abs(gap) < 1 << 40 and _layouts_overlap(gap, a.element_size(), a.shape, a.stride(), b.shape, b.stride()))


# ---------------------------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------------------------
PAIRINGS = {"adjacent": L.SQ_ROTARY_ADJACENT, "halves": L.SQ_ROTARY_HALVES}


def rotary(q, k, positions, axes, *, theta=10000.0, pairing="adjacent", norm_q=None, norm_k=None, eps=1e-6, out_q=None, out_k=None):
    """Rotary positions with several axes on q (B, T, Hq, D) and k (B, T, Hk, D), or packed (N, H, D) ones; k may be None.

    axes: the even widths of the axes' blocks inside a head, from column 0 on; columns behind the last block are not rotated.
    positions: int32 or float32 (T, A) or (B, T, A) with A = len(axes) (packed: (N, A)).  Pair i of axis a turns by
    position * theta ** (-2 i / axes[a]); pairing "adjacent" pairs columns (2i, 2i + 1) of a block, "halves" (i, i + width / 2).
    norm_q / norm_k: (D,) weights of the heads' RMS normalisation in front of the rotation, in q's dtype, both or neither.
    float32, float16 and bfloat16, D up to 256; arithmetic in fp32 (angles in fp64), rounded once.  out_q / out_k may be q / k
    themselves and overlap nothing else, themselves included.  No derivatives: inputs that want any are refused.  Returns (q, k) rotated; (q, None) without k."""
    global launch_count
    dev = q.get_device()
    if not q.is_cuda or not positions.is_cuda or not (k is None or k.is_cuda):
        _need_cuda(q, k, positions)
    if q.requires_grad or positions.requires_grad or (k is not None and k.requires_grad) or (norm_q is not None and norm_q.requires_grad) or \
            (norm_k is not None and norm_k.requires_grad):
        _no_grad(q, k, positions, norm_q, norm_k)
    if _forward_ad._current_level >= 0:
        _no_tangent(q, k, positions, norm_q, norm_k, out_q, out_k)
    if pairing not in PAIRINGS:
        raise ValueError(f"pairing must be one of {list(PAIRINGS)}")
    qs, dt, A = q.shape, q.dtype, len(axes)
    if len(qs) not in (3, 4) or (k is not None and (k.shape[:-2] != qs[:-2] or k.shape[-1] != qs[-1])):
        raise ValueError("rotary: q (B, T, Hq, D) and k (B, T, Hk, D), or packed (N, H, D) ones")
    if k is not None and (k.dtype != dt or k.get_device() != dev):
        raise TypeError("rotary: q and k must share dtype and device")
    if A == 0 or A > L.SQ_ROTARY_MAX_AXES:
        raise ValueError(f"rotary: 1 to {L.SQ_ROTARY_MAX_AXES} axes")
    B, T = (1, qs[0]) if len(qs) == 3 else qs[:2]
    D = qs[-1]
    ps = positions.shape
    if ps != (T, A) and ps != (B, T, A):
        raise ValueError(f"rotary: positions must be {(T, A)} or {(B, T, A)}, not {tuple(ps)}")
    if positions.dtype not in (torch.int32, torch.float32) or positions.get_device() != dev:
        raise TypeError("rotary: positions must be int32 or float32 on q's device")
    if (norm_k is not None and k is None) or (k is not None and (norm_q is None) != (norm_k is None)):
        raise ValueError("rotary: norm_q and norm_k come together, norm_k with k")
    positions = positions.contiguous()
    nq = nk = 0
    if norm_q is not None:
        for w in (norm_q, norm_k):
            if w is not None and (w.shape != (D,) or w.dtype != dt or w.get_device() != dev):
                raise ValueError("rotary: norm weights must be (D,) tensors of q's dtype on its device")
        norm_q = norm_q.contiguous()
        nq = norm_q.data_ptr()
        if norm_k is not None:
            norm_k = norm_k.contiguous()
            nk = norm_k.data_ptr()
    given = out_q is not None, out_k is not None and k is not None
    q, out_q, qi, qo = _rotary_pair(q, out_q, "q")
    if k is not None:
        k, out_k, ki, ko = _rotary_pair(k, out_k, "k")
        if (given[0] and _overlap(out_q, k)) or (given[1] and not (out_k is k and out_q is q) and _overlap(out_k, q)) or \
                (given[0] and given[1] and not (out_k is k or out_q is q) and _overlap(out_q, out_k)):
            raise ValueError("rotary: an output overlaps the other tensor")
        a = (q.data_ptr(), k.data_ptr(), out_q.data_ptr(), out_k.data_ptr(), _dt(q), PAIRINGS[pairing], B, T, qs[-2], k.shape[-2])
    elif out_k is not None:
        raise ValueError("rotary: out_k without k")
    else:
        ki = ko = (0, 0, 0)
        a = (q.data_ptr(), 0, out_q.data_ptr(), 0, _dt(q), PAIRINGS[pairing], B, T, qs[-2], 0)
    a = _ROTARY.pack(*a, D, A, struct.pack(f"{A}i", *axes), *qi, *ki, *qo, *ko, positions.data_ptr(), T * A if len(ps) == 3 else 0, A,
                     1 if positions.dtype == torch.float32 else 0, eps, theta, nq, nk)
    _run(L.load().sq_rotary_packed, "sq_rotary", dev, a)
    if q.numel():
        launch_count += 1
    return out_q, out_k


def _rotary_pair(x, out, name):
    """(input, output, their (batch, token, head) strides)"""
    xs = x.stride()
    if xs[-1] != 1 and x.numel():
        if out is x:
            raise ValueError("rotary: in place needs a contiguous last dimension")
        x = x.contiguous()
        xs = x.stride()
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    else:
        if out is not x and (out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or out.stride(-1) != 1):
            raise ValueError(f"rotary: out_{name} must have {name}'s shape, dtype and device and a contiguous last dimension")
        same = out is x or (out.data_ptr() == x.data_ptr() and all(n == 1 or a == b for n, a, b in zip(x.shape, out.stride(), xs)))
        if _overlaps_itself(out) or (not same and _overlap(out, x)):
            raise ValueError(f"rotary: out_{name} overlaps itself, or {name} without being the same elements")
    os = out.stride()
    return (x, out, xs[:3], os[:3]) if len(xs) == 4 else (x, out, (0, xs[0], xs[1]), (0, os[0], os[1]))


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
def _no_grad(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("segquant_b200: this operator has no backward pass; detach its inputs or run it under torch.no_grad()")


def _no_tangent(*tensors):
    """Called inside a forward-mode level only: elsewhere no tensor has a tangent."""
    if any(t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("segquant_b200: this operator has no derivative; its inputs may not carry tangents")


def _tma_view(t):
    """t itself where the kernel can read it in place (last dimension contiguous, other strides positive multiples of 16
    bytes, 16-byte aligned), else a contiguous copy."""
    st = t.stride()
    if st[-1] == 1 and t.data_ptr() % 16 == 0 and (t.is_contiguous() and st[-2] % 8 == 0 or
                                                   all(n <= 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:-1], st[:-1]))):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _int32_list(t, n, name, dev):
    if t.dtype != torch.int32 or t.shape != (n,) or t.get_device() != dev or not t.is_cuda:
        raise ValueError(f"attention: {name} must be an int32 tensor of {n} elements on cuda:{dev}")
    return t.contiguous()


def attention(q, k, v, *, causal=False, scale=None, q_offsets=None, kv_offsets=None, q_lens=None, kv_lens=None, out=None,
              return_lse=False):
    """softmax(scale * q k^T) v for 16-bit tensors, statistics in fp32; scale defaults to D ** -0.5.

    Sequences of one extent: q (B, Tq, Hq, D), k and v (B, Tk, Hkv, D), Hq a multiple of Hkv (query head h reads key head
    h // (Hq // Hkv)); q_lens / kv_lens (int32 (B,), on the device) give the valid tokens of each where they are fewer.
    Packed sequences: q (Nq, Hq, D), k and v (Nk, Hkv, D) with q_offsets (int32 (B + 1,), non-decreasing, on the device);
    kv_offsets defaults to q_offsets.  D is a multiple of 8 up to 128; strides are free as long as D is contiguous (views
    that the loads cannot read in place are copied first).

    causal: query i of a sequence sees its keys below i + 1 + kv_len - q_len, so its last query sees its last key.  A
    query that sees no key gets 0 (lse -inf).  Rows that belong to no sequence are 0 in a new result and left alone in
    `out`, which has q's shape and dtype, D contiguous, strides and address multiples of 16 bytes, and overlaps neither itself nor an input.
    No derivatives: inputs that want any are refused.
    return_lse: also the float32 logarithm of the row sums, (B, Tq, Hq) or (Nq, Hq)."""
    global launch_count
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        _need_cuda(q, k, v)
    if q.requires_grad or k.requires_grad or v.requires_grad:
        _no_grad(q, k, v)
    if _forward_ad._current_level >= 0:
        _no_tangent(q, k, v, out)
    packed = q_offsets is not None
    if kv_offsets is not None and not packed:
        raise ValueError("attention: kv_offsets needs q_offsets")
    if packed and (q_lens is not None or kv_lens is not None):
        raise ValueError("attention: packed sequences have offsets, not lengths")
    dt, qs, ks = q.dtype, q.shape, k.shape
    if dt not in (torch.bfloat16, torch.float16) or k.dtype != dt or v.dtype != dt:
        raise TypeError("attention: q, k and v must share a 16-bit dtype")
    rank = 3 if packed else 4
    if len(qs) != rank or len(ks) != rank or v.shape != ks or ks[-1] != qs[-1] or (not packed and ks[0] != qs[0]):
        raise ValueError("attention: q (B, Tq, Hq, D) with k, v (B, Tk, Hkv, D), or packed q (Nq, Hq, D) with k, v (Nk, Hkv, D)")
    dev = q.get_device()
    if k.get_device() != dev or v.get_device() != dev:
        raise ValueError("attention: q, k and v must be on one device")
    Tq, Hq, D = qs[-3:]
    Tk, Hkv = ks[-3:-1]
    if Hkv == 0 or Hq % Hkv:
        raise ValueError(f"attention: {Hq} query heads do not share {Hkv} key heads evenly")
    if D % 8 or not 8 <= D <= L.SQ_ATTENTION_MAX_D:
        raise ValueError(f"attention: head width {D} is not a multiple of 8 up to {L.SQ_ATTENTION_MAX_D}")
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError("attention: scale must be positive and finite")
    if packed:
        kv_offsets = q_offsets if kv_offsets is None else kv_offsets
        B = q_offsets.numel() - 1
        if B < 0:
            raise ValueError("attention: q_offsets needs at least one element")
        q_offsets, kv_offsets = _int32_list(q_offsets, B + 1, "q_offsets", dev), _int32_list(kv_offsets, B + 1, "kv_offsets", dev)
    else:
        B = qs[0]
        if q_lens is not None:
            q_lens = _int32_list(q_lens, B, "q_lens", dev)
        if kv_lens is not None:
            kv_lens = _int32_list(kv_lens, B, "kv_lens", dev)
    fill_rest = out is None
    if fill_rest:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _need_cuda(out)
        if out.shape != qs or out.dtype != dt or out.device != q.device or _tma_view(out) is not out:
            raise ValueError("attention: out must have q's shape, dtype and device, a contiguous last dimension, and strides and address in "
                             "multiples of 16 bytes")
        if _overlaps_itself(out) or _overlap(out, q) or _overlap(out, k) or _overlap(out, v):
            raise ValueError("attention: out overlaps itself or an input")
    lse = torch.full(qs[:-1], float("-inf"), dtype=torch.float32, device=q.device) if return_lse else None
    if packed and B == 0:
        if fill_rest:
            out.zero_()
    elif q.numel():
        qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
        if (qp | kp | vp) & 15 or not (q.is_contiguous() and k.is_contiguous() and v.is_contiguous()):
            q, k, v = _tma_view(q), _tma_view(k), _tma_view(v)
            qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
        sq, sk, sv, so = q.stride(), k.stride(), v.stride(), out.stride()
        if packed:                                     # no batch stride
            strides = (0, sq[0], sq[1], 0, sk[0], sk[1], 0, sv[0], sv[1], 0, so[0], so[1])
        else:
            strides = (*sq[:3], *sk[:3], *sv[:3], *so[:3])
        head = (qp, kp, vp, out.data_ptr(), lse.data_ptr() if return_lse else 0, _DT[dt], 1 if causal else 0, B, Tq, Tk, Hq, Hkv, D, 1 if fill_rest else 0,
                *strides, q_offsets.data_ptr() if packed else 0, kv_offsets.data_ptr() if packed else 0,
                q_lens.data_ptr() if q_lens is not None else 0, kv_lens.data_ptr() if kv_lens is not None else 0, scale, 0)
        lib, a = L.load(), _ATTENTION.pack(*head, 0, 0)
        need = lib.sq_attention_scratch_bytes_packed(a)
        if need < 0:
            L.check(need, "sq_attention_scratch_bytes")
        if need:
            scratch = q.new_empty(need, dtype=torch.uint8)
            a = _ATTENTION.pack(*head, scratch.data_ptr(), need)
        _run(lib.sq_attention_packed, "sq_attention", dev, a)
        launch_count += 2 if need else 1
    return (out, lse) if return_lse else out


# ---------------------------------------------------------------------------------------------
# weights
# ---------------------------------------------------------------------------------------------
def quantize_weight(w, out, scale, out_kind, group_size=0):
    """real_quantized_quantize_weights(weights, outputs, scale_w): scale is a python float, a
    (N,) tensor or, with group_size, a (N, K/group_size) tensor.  Writes into `out`."""
    global launch_count
    _need_cuda(w, out)
    if w.dim() != 2:
        raise ValueError("weights must be [N, K]")
    w = w.contiguous()
    N, K = w.shape
    if isinstance(scale, torch.Tensor):
        sc = _f32(scale, w.device)
        if group_size and sc.dim() == 2:
            mode = 2
            if sc.shape != (N, K // group_size):
                raise ValueError(f"group scale shape {tuple(sc.shape)} != {(N, K // group_size)}")
        else:
            mode = 1
            if sc.numel() != N:
                raise ValueError(f"per-channel scale has {sc.numel()} elements, expected {N}")
        scalar, ptr = 0.0, sc.data_ptr()
    else:
        mode, scalar, ptr, sc = 0, float(scale), None, None
    with torch.cuda.device(w.device):
        L.check(L.load().sq_quantize_weight(w.data_ptr(), _dt(w), N, K, mode, scalar, ptr, int(group_size or 0), out_kind,
                                            out.data_ptr(), _stream(w)), "sq_quantize_weight")
    launch_count += 1
    return out


def unpack_int4(packed, numel=None):
    global launch_count
    _need_cuda(packed)
    packed = packed.contiguous()
    numel = packed.numel() * 2 if numel is None else numel
    out = torch.empty(numel, dtype=torch.int8, device=packed.device)
    with torch.cuda.device(packed.device):
        L.check(L.load().sq_unpack_int4(packed.data_ptr(), out.data_ptr(), numel, _stream(packed)), "sq_unpack_int4")
    launch_count += 1
    return out


# ---------------------------------------------------------------------------------------------
# GEMM
# ---------------------------------------------------------------------------------------------
def num_units(bounds, group_size=0):
    arr = (ctypes.c_int32 * len(bounds))(*[int(b) for b in bounds])
    return L.check(L.load().sq_gemm_num_units(len(bounds) - 1, arr, int(group_size or 0)), "sq_gemm_num_units")


def gemm(kind, xq, wq, N, bounds, sx, sw, *, xq_neg=None, sx_neg=None, per_token=False, group_size=0,
         sw_strides=(0, 0, 0, 1), bias=None, out_dtype=torch.float32, out=None, x_batched=True, w_seg_as_batch=False,
         y_strides=None, sx_batch_stride=None, want_acc=False, peer_outputs=None):
    """xq: (B, M, K) uint8 contiguous (or B == 1 shared by `batch` problems when x_batched=False).

    wq: weights, (Bw, N, K) bytes or (Bw, N, K/2) packed int4, contiguous.
    sw_strides = (batch, segment, group, column) element strides into `sw`."""
    global launch_count
    _need_cuda(xq, wq, sx, sw, bias)
    Bx, M, K = xq.shape
    Bw = wq.shape[0]
    batch = 1 if w_seg_as_batch else max(Bx, Bw)
    S = len(bounds) - 1
    w4 = kind == L.SQ_GEMM_W4A8
    if sw.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("weight scales must be float32 or bfloat16")
    if S > L.SQ_MAX_SEGS:
        raise L.SegQuantError(L.SQ_ERR_INVALID_ARG, f"at most {L.SQ_MAX_SEGS} segments per call, got {S}")
    bounds = [*map(int, bounds)]
    try:
        packed_bounds = struct.pack(f"{S + 1}i", *bounds)
    except struct.error:
        raise L.SegQuantError(L.SQ_ERR_INVALID_ARG, f"segment bounds past 32 bits: {bounds}") from None
    Kw = (bounds[1] - bounds[0]) if w_seg_as_batch else K
    w_row = Kw // 2 if w4 else Kw
    sx_strides = (S * M, M, 1) if per_token else (S, 1, 0)
    y = out if out is not None else xq.new_empty((batch, M, N), dtype=out_dtype)
    y_bs, y_rs = y_strides if y_strides is not None else (M * N, N)
    acc, peers, n_peers, prs, pco = None, _NO_PEERS, 0, 0, 0
    if peer_outputs is not None:
        # fused all-gather: (device pointers of the peers' [M, *] buffers, row stride, column offset) in elements
        ptrs, prs, pco = peer_outputs
        n_peers = len(ptrs)
        if n_peers > L.SQ_MAX_PEERS:
            raise ValueError(f"at most {L.SQ_MAX_PEERS} peer outputs")
        peers = (*(int(ptr) for ptr in ptrs), *_NO_PEERS[n_peers:])
    if want_acc:
        units = num_units(bounds, group_size)
        sides = 2 if xq_neg is not None else 1
        acc = torch.zeros((batch, units, sides, M, N), dtype=torch.int32, device=xq.device)
    a = _GEMM.pack(
        kind, _DT[out_dtype], batch, M, N, K,
        xq.data_ptr(), xq_neg.data_ptr() if xq_neg is not None else 0, M * K if (x_batched and Bx > 1) else 0, K,
        wq.data_ptr(), N * w_row if Bw > 1 else 0, w_row, 1 if w_seg_as_batch else 0,
        S, packed_bounds, int(group_size or 0), 1 if sw.dtype == torch.bfloat16 else 0,
        sx.data_ptr(), sx_neg.data_ptr() if sx_neg is not None else 0,
        sx_strides[0] if sx_batch_stride is None else sx_batch_stride, sx_strides[1], sx_strides[2],
        sw.data_ptr(), *sw_strides,
        bias.data_ptr() if bias is not None else 0, _dt(bias) if bias is not None else 0, 0, 0,
        y.data_ptr(), y_bs, y_rs, acc.data_ptr() if acc is not None else 0, n_peers, 0, *peers, int(prs), int(pco))
    _run(L.load().sq_gemm_packed, "sq_gemm", xq.get_device(), a)
    launch_count += 1
    return (y, acc) if want_acc else y


def device_status():
    """Synchronise and return the word kernels write when a bounded wait gave up (0 = fine)."""
    return int(L.load().sq_device_status())


def push_columns(block, peer_ptrs, peer_row_stride_bytes):
    """Copy the 2-D view `block` ([rows, width], a column block inside this rank's result matrix, last dim contiguous) to
    the device addresses peer_ptrs (the block's position inside each peer GPU's matrix, mapped into this process)."""
    global launch_count
    _need_cuda(block)
    if block.dim() != 2 or block.stride(1) != 1:
        raise ValueError("push_columns needs a [rows, width] view with a contiguous last dim")
    if not peer_ptrs:
        return
    esz = block.element_size()
    arr = (ctypes.c_void_p * len(peer_ptrs))(*[int(p) for p in peer_ptrs])
    with torch.cuda.device(block.device):
        L.check(L.load().sq_push_columns(block.data_ptr(), block.shape[0], block.shape[1] * esz, block.stride(0) * esz, len(peer_ptrs),
                                         arr, int(peer_row_stride_bytes), _stream(block)), "sq_push_columns")
    launch_count += 1


def peer_barrier(rank, flag_ptrs, epoch, device):
    """Stream-ordered barrier over flag words in peer-mapped memory (sq_peer_barrier): flag_ptrs[j] = device address of
    rank j's array of len(flag_ptrs) uint32 words, epoch = number of this collective call (1, 2, ...)."""
    global launch_count
    world = len(flag_ptrs)
    if world == 1:
        return
    arr = (ctypes.c_void_p * world)(*[int(p) for p in flag_ptrs])
    with torch.cuda.device(device):
        L.check(L.load().sq_peer_barrier(int(rank), world, arr, int(epoch) & 0xFFFFFFFF,
                                         ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)), "sq_peer_barrier")
    launch_count += 1


def check_device():
    """Synchronise and raise SegQuantError(SQ_ERR_DEVICE_TIMEOUT) if a kernel reported a bounded wait that ran out."""
    L.check(L.load().sq_check_device(), "sq_check_device")


def set_gemm_schedule(bn=0, two_cta=-1, ksub=0, no_gemv=0):
    """Force the GEMM schedule process-wide (0 / -1 = automatic); results do not depend on it.  Test and tuning aid."""
    L.check(L.load().sq_set_gemm_schedule(int(bn), int(two_cta), int(ksub), int(no_gemv)), "sq_set_gemm_schedule")


# ---------------------------------------------------------------------------------------------
# fused layer forward
# ---------------------------------------------------------------------------------------------
def seg_linear(kernel_type, x, wq, N, bounds, sx, sw, *, sx_neg=None, dynamic=False, group_size=0,
               sw_strides=(0, 0, 0, 1), bias=None, smooth=None, w_seg_as_batch=False, out_dtype=None, out=None,
               peer_outputs=None):
    """SegmentLinear.forward on the real-quant path in two launches: quantise x [.., K] with the
    per-K-segment (or DualScale, or dynamic per-token) scales, then one GEMM that sums the
    segments in fp32 registers, adds the bias and casts.  Returns [.., N] in x.dtype."""
    kind, a_kind, _ = KERNELS[kernel_type]
    lead = x.shape[:-1]
    K = x.shape[-1]
    out_dtype = out_dtype or x.dtype
    dual = sx_neg is not None
    if out is not None:
        # write straight into a caller-provided (B, M, N) view (any batch / row stride, N contiguous), e.g. a slice of
        # a joint token buffer: one problem per batch entry, all sharing the weight matrix
        if dynamic or x.dim() != 3 or out.dim() != 3 or out.stride(-1) != 1 or out.shape[:2] != x.shape[:2] or out.shape[2] != N:
            raise ValueError("out= needs a static-scale (B, M, K) input and a (B, M, N) output view with a contiguous last dim")
        xq, xqn = quantize_act(x if x.stride(-1) == 1 else x.contiguous(), bounds, sx, sx_neg, a_kind, smooth=smooth, shared_scales=True)
        gemm(kind, xq, wq, N, bounds, sx, sw, xq_neg=xqn, sx_neg=sx_neg, group_size=group_size, sw_strides=sw_strides, bias=bias,
             out_dtype=out.dtype, out=out, y_strides=(out.stride(0), out.stride(1)), sx_batch_stride=0, w_seg_as_batch=w_seg_as_batch,
             peer_outputs=peer_outputs)
        return out
    if peer_outputs is not None:
        raise ValueError("peer_outputs needs out= (a (1, M, N) view of this rank's own buffer)")
    if x.dim() == 3 and x.stride(-1) == 1 and not x.is_contiguous() and not dynamic:
        # a strided (B, M, K) view (e.g. a token slice of a joint sequence): the quantise kernel reads it
        # in place and writes contiguous bytes, so no copy of x is made
        xq, xqn = quantize_act(x, bounds, sx, sx_neg, a_kind, smooth=smooth, shared_scales=True)
        rows = xq.shape[0] * xq.shape[1]
        y = gemm(kind, xq.view(1, rows, K), wq, N, bounds, sx, sw, xq_neg=None if xqn is None else xqn.view(1, rows, K),
                 sx_neg=sx_neg, group_size=group_size, sw_strides=sw_strides, bias=bias, out_dtype=out_dtype,
                 w_seg_as_batch=w_seg_as_batch)
        return y.reshape(*lead, N)
    x2 = x.reshape(-1, K)
    if dynamic:
        xq, xqn, sxd, sxnd = quantize_act_dynamic(x2, bounds, a_kind, dual=dual, smooth=smooth)
        y = gemm(kind, xq.unsqueeze(0), wq, N, bounds, sxd, sw, xq_neg=xqn, sx_neg=sxnd, per_token=True,
                 group_size=group_size, sw_strides=sw_strides, bias=bias, out_dtype=out_dtype,
                 w_seg_as_batch=w_seg_as_batch)
    else:
        xq, xqn = quantize_act(x2, bounds, sx, sx_neg, a_kind, smooth=smooth)
        y = gemm(kind, xq, wq, N, bounds, sx, sw, xq_neg=xqn, sx_neg=sx_neg, group_size=group_size,
                 sw_strides=sw_strides, bias=bias, out_dtype=out_dtype, w_seg_as_batch=w_seg_as_batch)
    return y.reshape(*lead, N)


# ---------------------------------------------------------------------------------------------
# the reference's pybind functions
# ---------------------------------------------------------------------------------------------
def _segment_batches(inputs):
    """Classify the (S, ..., M, K) input of the reference contract without copying it.
    Returns (x3 (B, M, K) view, shared) where shared=True means all S batches are the same
    (a stride-0 expand, segquant/layers/segment_tensor_manager.py:21-23)."""
    S, K = inputs.shape[0], inputs.shape[-1]
    if inputs.stride(0) == 0 and S >= 1:
        first = inputs[0]
        first = first.reshape(-1, K) if first.is_contiguous() else first.contiguous().view(-1, K)
        return first.unsqueeze(0), True
    if inputs.dim() == 3 and inputs.stride(-1) == 1:
        return inputs, False  # (S, M, K) with arbitrary batch / row stride: the kernel takes it as is
    if inputs.dim() > 3 and inputs.stride(-1) == 1:
        try:
            return inputs.view(S, -1, K), False
        except RuntimeError:
            pass
    return inputs.contiguous().view(S, -1, K), False


def real_quantized_gemm_scaled(kernel_type, inputs, weights, scale_x, scale_w, neg_scale_x=None):
    """`{P}_real_quantized_gemm_scaled(inputs, weights, scale_x, scale_w)` and, when neg_scale_x is
    given (scale_x then being the positive scale), `{P}_real_quantized_gemm_dual_scaled`.

    inputs (S, ..., M, K) float; weights (S, N, K) int8 / uint8-as-e4m3 or (S, N*K/2) packed int4;
    scales float32 with S or S*M (x) and S or S*N (w) elements.  Returns a new (S, ..., M, N)
    tensor in the input dtype, un-summed and without bias (real_gemm.cu:644-687)."""
    kind, a_kind, _ = KERNELS[kernel_type]
    _need_cuda(inputs, weights)
    S, K = inputs.shape[0], inputs.shape[-1]
    lead = tuple(inputs.shape[1:-1])
    x3, shared = _segment_batches(inputs)
    M = x3.shape[1]
    if weights.shape[0] != S:
        raise RuntimeError(f"weights have {weights.shape[0]} segments, inputs {S}")
    weights = weights.contiguous()
    if kind == L.SQ_GEMM_W4A8:
        N = weights.shape[1] * 2 // K   # real_gemm.cu:670
        w3 = weights.view(S, N, K // 2)
    else:
        N = weights.shape[1]
        w3 = weights.view(S, N, K)
    dev = inputs.device
    sx = _f32(scale_x, dev).reshape(-1)
    sxn = _f32(neg_scale_x, dev).reshape(-1) if neg_scale_x is not None else None
    sw = _f32(scale_w, dev).reshape(-1)
    per_token = sx.numel() != S          # real_gemm.cu:703
    if per_token and sx.numel() != S * M:
        raise RuntimeError(f"scale_x has {sx.numel()} elements, expected {S} or {S * M}")
    w_scalar = sw.numel() == S           # real_gemm.cu:743
    if not w_scalar and sw.numel() != S * N:
        raise RuntimeError(f"scale_w has {sw.numel()} elements, expected {S} or {S * N}")
    sw_strides = (1, 0, 0, 0) if w_scalar else (N, 0, 0, 1)
    bounds = [0, K]
    if shared:
        # a stride-0 expand: every batch re-reads the same rows (its scales may differ), nothing is copied
        x3 = x3.expand(S, M, K)
    xq, xqn = quantize_act(x3, bounds, sx, sxn, a_kind, per_token=per_token)
    y = gemm(kind, xq, w3, N, bounds, sx, sw, xq_neg=xqn, sx_neg=sxn, per_token=per_token, sw_strides=sw_strides,
             out_dtype=inputs.dtype)
    return y.view(S, *lead, N)
