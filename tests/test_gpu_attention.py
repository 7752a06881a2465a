"""GPU: ops.attention against softmax(scale q k^T) v in fp64.

Tolerance, element by element, with u = finfo.eps / 2 (half a step of the 16-bit type) and A = sum_j p_j |v_j| of that element:
the result is rounded once (u |o|), every p is rounded once before the second product (u A), and what fp32 adds: a score is off
by at most D 2^-23 sum |q k| scale (a sum of D products) + 2^-23 |s| (its product with scale log2 e and the subtraction of the
maximum), an exponential by 4e-6 (2^-22 of the special function, 3e-6 of the polynomial), so p and the row sum by
eta = the three together, each, and the second product by n 2^-23 A for n keys:  A (u + 2 eta + n 2^-23) + u |o|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from segquant_b200 import ops

DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def _rand(gen, *shape, dtype=BF, mul=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * mul).to(dtype)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _reference(q, k, v, causal, scale):
    """(o, lse, tolerance of o, tolerance of lse) of one sequence in fp64: q (tq, hq, d), k and v (tk, hkv, d)."""
    tq, hq, d = q.shape
    tk, hkv, _ = k.shape
    u = torch.finfo(q.dtype).eps / 2
    if tk == 0:
        z = torch.zeros(tq, hq, d, dtype=torch.float64, device=q.device)
        return z, z[..., 0] - math.inf, z, z[..., 0]
    q, k, v = (t.double().transpose(0, 1) for t in (q, k, v))
    k, v = k.repeat_interleave(hq // hkv, 0), v.repeat_interleave(hq // hkv, 0)
    s = q @ k.transpose(1, 2) * scale
    sabs = (q.abs() @ k.abs().transpose(1, 2)).amax(dim=-1) * scale
    if causal:
        i = torch.arange(tq, device=q.device)[:, None] + tk - tq
        s = s.masked_fill(torch.arange(tk, device=q.device)[None] > i, -math.inf)
    lse = torch.logsumexp(s, dim=-1)
    some = torch.isfinite(lse)[..., None]
    p = torch.where(some, torch.exp(s - lse[..., None]), 0.0)
    o, a = p @ v, p @ v.abs()
    eta = (d * 2.0 ** -23 + 2.0 ** -23 * 1.5) * sabs + 4e-6
    tol = a * (u + 2 * eta[..., None] + tk * 2.0 ** -23) + u * o.abs() + 1e-30
    return o.transpose(0, 1), lse.transpose(0, 1), tol.transpose(0, 1), (eta + tk * 2.0 ** -24 + 2.0 ** -22 * lse.abs().nan_to_num(0, 0, 0)).transpose(0, 1)


def _check(got, lse, want, what=""):
    o, l, tol, ltol = want
    err = (got.double() - o).abs()
    assert torch.isfinite(got).all(), what
    assert (err <= tol).all(), (what, float((err / tol).nan_to_num(0).max()))
    if lse is not None:
        none = l == -math.inf
        assert torch.equal(lse == -math.inf, none), what
        assert (((lse.double() - l).abs() <= ltol) | none).all(), (what, float(((lse.double() - l).abs() / ltol).nan_to_num(0).max()))


def _batched(q, k, v, causal=False, scale=None, q_lens=None, kv_lens=None, **kw):
    """Runs and checks; the rows behind a sequence's queries have to be 0."""
    out, lse = ops.attention(q, k, v, causal=causal, scale=scale, return_lse=True, **kw,
                             q_lens=None if q_lens is None else torch.tensor(q_lens, dtype=torch.int32, device=DEV),
                             kv_lens=None if kv_lens is None else torch.tensor(kv_lens, dtype=torch.int32, device=DEV))
    for i in range(q.shape[0]):
        a, b = q.shape[1] if q_lens is None else q_lens[i], k.shape[1] if kv_lens is None else kv_lens[i]
        _check(out[i, :a], lse[i, :a], _reference(q[i, :a], k[i, :b], v[i, :b], causal, scale or q.shape[-1] ** -0.5), i)
        assert not out[i, a:].any() and (lse[i, a:] == -math.inf).all()
    assert ops.device_status() == 0
    return out


SHAPES = [  # batch, tq, tk, hq, hkv, d, causal
    (1, 1, 1, 1, 1, 8, False), (1, 128, 128, 1, 1, 64, False), (1, 129, 127, 2, 1, 64, False), (2, 257, 300, 3, 3, 64, True), (1, 256, 256, 2, 2, 128, True),
    (2, 300, 777, 4, 2, 128, False), (1, 77, 1000, 10, 2, 80, True), (1, 1000, 1000, 4, 4, 96, True), (1, 640, 640, 2, 1, 72, True), (1, 200, 130, 7, 1, 48, False),
    (1, 500, 40, 2, 2, 64, True),       # causal with fewer keys than queries: the first rows see nothing
    (1, 20, 1500, 33, 1, 64, True),     # 33 heads of one key head
    (1, 3, 65, 64, 2, 32, True), (1, 30, 5000, 4, 4, 128, True),      # few tiles: the keys in parts
    # few rows against many keys
    (1, 1, 33, 2, 1, 64, True), (3, 1, 1531, 24, 8, 64, True), (2, 4, 3000, 8, 2, 128, True), (1, 3, 700, 5, 1, 80, True), (2, 2, 100, 6, 3, 72, False),
    (1, 16, 999, 2, 2, 128, True), (1, 5, 3, 2, 2, 64, True), (1, 1, 31, 16, 1, 8, False), (1, 2, 5000, 8, 1, 120, True),
]


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_batched_against_fp64(native_lib, shape, dtype):
    b, tq, tk, hq, hkv, d, causal = shape
    g = _gen(1)
    _batched(_rand(g, b, tq, hq, d, dtype=dtype, mul=1.5), _rand(g, b, tk, hkv, d, dtype=dtype), _rand(g, b, tk, hkv, d, dtype=dtype), causal)


def test_many_blocks_to_a_slot(native_lib):
    """Parts of several ring lengths, many CTAs at once, several times: a block's wait must not pass on the one before it."""
    g = _gen(2)
    q, k, v = _rand(g, 40, 1, 32, 128), _rand(g, 40, 2000, 8, 128), _rand(g, 40, 2000, 8, 128)
    first = _batched(q, k, v, True)
    for _ in range(5):
        assert torch.equal(ops.attention(q, k, v, causal=True), first)
    q, k, v = _rand(g, 150, 1, 4, 64), _rand(g, 150, 1100, 4, 64), _rand(g, 150, 1100, 4, 64)
    first = _batched(q, k, v, True)
    for _ in range(5):
        assert torch.equal(ops.attention(q, k, v, causal=True), first)


@pytest.mark.parametrize("tq,hq,hkv,d", [(1, 8, 2, 128), (1, 3, 3, 64), (70, 4, 2, 64), (300, 2, 2, 128)], ids=str)
@pytest.mark.parametrize("causal", [False, True])
def test_lengths_with_nan_behind_them(native_lib, tq, hq, hkv, d, causal):
    """A padded batch and caches that are not full: lengths of zero and one and of whole tiles, NaN and infinities behind them."""
    g = _gen(3)
    kv_lens, q_lens = [0, 1, 31, 32, 128, 129, 700, 257], [0, 1, tq, max(tq - 1, 0), tq, tq // 2, tq, tq]
    q, k, v = _rand(g, 8, tq, hq, d), _rand(g, 8, 700, hkv, d), _rand(g, 8, 700, hkv, d)
    for i, (a, b) in enumerate(zip(q_lens, kv_lens)):
        q[i, a:] = math.nan
        k[i, b:] = math.inf if i % 2 else math.nan
        v[i, b:] = math.nan if i % 2 else -math.inf
    _batched(q, k, v, causal, q_lens=q_lens, kv_lens=kv_lens)
    _batched(q[:, :, :, :], k, v, causal, kv_lens=kv_lens) if tq == 1 and torch.isfinite(q).all() else None
    # lengths outside the tensors are clamped
    big = torch.tensor([5000] * 8, dtype=torch.int32, device=DEV)
    fin_q, fin_k, fin_v = (t.nan_to_num(0.5, 0.5, -0.5) for t in (q, k, v))
    assert torch.equal(ops.attention(fin_q, fin_k, fin_v, q_lens=big, kv_lens=big), ops.attention(fin_q, fin_k, fin_v))
    assert not ops.attention(fin_q, fin_k, fin_v, kv_lens=-big).any()


def _packed_case(lens, kv_lens, hq, hkv, d, dtype=BF, lead=0, trail=0, seed=4):
    g = _gen(seed)
    qo = torch.tensor([lead] + lens).cumsum(0)
    ko = torch.tensor([lead] + kv_lens).cumsum(0)
    q = _rand(g, int(qo[-1]) + trail, hq, d, dtype=dtype, mul=1.5)
    k, v = _rand(g, int(ko[-1]) + trail, hkv, d, dtype=dtype), _rand(g, int(ko[-1]) + trail, hkv, d, dtype=dtype)
    return q, k, v, qo.tolist(), ko.tolist()


PACKED = [
    ([5], [5], 1, 1, 64), ([1, 1, 1], [1, 1, 1], 2, 2, 64), ([517, 1, 0, 333, 0, 77, 130], [517, 1, 0, 333, 0, 77, 130], 4, 2, 128),
    ([64, 200, 7], [1064, 3300, 84], 10, 2, 80), ([300, 2, 40], [10, 0, 40], 2, 1, 64), ([0, 0], [0, 0], 2, 2, 64), ([1] * 70, list(range(70)), 8, 2, 64),
    ([1, 2, 0, 3, 1], [900, 33, 5, 128, 1], 6, 2, 128), ([2000], [2000], 2, 2, 128), ([100] * 40, [100] * 40, 1, 1, 32),
]


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("case", range(len(PACKED)))
def test_packed_against_fp64(native_lib, case, causal, dtype):
    lens, kv_lens, hq, hkv, d = PACKED[case]
    q, k, v, qo, ko = _packed_case(lens, kv_lens, hq, hkv, d, dtype, lead=3, trail=9)
    for a, b in ((q, qo), (k, ko), (v, ko)):                     # tokens of no sequence
        a[:3], a[b[-1]:] = math.nan, math.inf
    offs = [torch.tensor(t, dtype=torch.int32, device=DEV) for t in (qo, ko)]
    out, lse = ops.attention(q, k, v, causal=causal, q_offsets=offs[0], kv_offsets=offs[1], return_lse=True)
    kept = torch.full_like(q, 7.0)
    assert ops.attention(q, k, v, causal=causal, q_offsets=offs[0], kv_offsets=offs[1], out=kept) is kept
    for i in range(len(lens)):
        s, t = slice(qo[i], qo[i + 1]), slice(ko[i], ko[i + 1])
        _check(out[s], lse[s], _reference(q[s], k[t], v[t], causal, d ** -0.5), i)
        assert torch.equal(kept[s], out[s])
    for rest in (slice(0, qo[0]), slice(qo[-1], None)):          # rows of no sequence: 0 in a new result, left alone in one that is given
        assert not out[rest].any() and (kept[rest] == 7.0).all() and (lse[rest] == -math.inf).all()
    assert ops.device_status() == 0


def test_one_sequence_never_reaches_another(native_lib):
    q, k, v, qo, ko = _packed_case([100, 140, 90], [100, 140, 90], 2, 2, 64)
    offs = torch.tensor(qo, dtype=torch.int32, device=DEV)
    clean = ops.attention(q, k, v, q_offsets=offs)
    for t in (q, k, v):
        t[100:240] = math.nan
    dirty = ops.attention(q, k, v, q_offsets=offs)
    assert torch.equal(clean[:100], dirty[:100]) and torch.equal(clean[240:], dirty[240:]) and torch.isnan(dirty[100:240]).all()


@pytest.mark.parametrize("tq", [1, 40, 300])
def test_layouts(native_lib, tq):
    g = _gen(6)
    buf = _rand(g, 2, tq, 3, 4, 64)                              # q | k | v side by side
    q, k, v = buf.unbind(2)
    want = ops.attention(q.contiguous(), k.contiguous(), v.contiguous(), causal=True)
    _batched(q, k, v, True)
    assert torch.equal(ops.attention(q, k, v, causal=True), want)
    heads_first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    assert torch.equal(ops.attention(heads_first(q), heads_first(k), v, causal=True), want)
    odd = torch.empty(2 * tq * 4 * 64 + 1, dtype=BF, device=DEV)[1:].view(2, tq, 4, 64)          # 2 bytes off: copied
    assert torch.equal(ops.attention(odd.copy_(q), k, v, causal=True), want)
    wide = torch.empty(2, tq, 4, 67, dtype=BF, device=DEV)[..., :64]                              # strides of 67: copied
    assert torch.equal(ops.attention(q, wide.copy_(k), v, causal=True), want)
    last = torch.empty(2, tq, 64, 4, dtype=BF, device=DEV).transpose(2, 3)                        # columns apart: copied
    assert torch.equal(ops.attention(q, k, last.copy_(v), causal=True), want)
    one = k[:, :, :1].expand(-1, -1, 4, -1)                                                        # one head for all: copied
    assert torch.equal(ops.attention(q, one, v, causal=True), ops.attention(q, one.contiguous(), v, causal=True))
    out = torch.full((2, tq, 3, 4, 64), 5.0, dtype=BF, device=DEV)
    ops.attention(q, k, v, causal=True, out=out[:, :, 1])
    assert torch.equal(out[:, :, 1], want) and (out[:, :, 0] == 5.0).all() and (out[:, :, 2] == 5.0).all()


def test_extreme_scores(native_lib):
    g = _gen(7)
    for tq in (1, 200):
        q, k, v = _rand(g, 1, tq, 2, 64), _rand(g, 1, 300, 2, 64), _rand(g, 1, 300, 2, 64)
        _batched(q, k, v, scale=60.0)                            # one key has all the weight
        _batched(q, k, v, scale=1e-6)                            # all keys the same
        _batched(q * 0, k, v)
        rising = k * 0 + torch.linspace(-8, 8, 300, device=DEV).view(1, 300, 1, 1).to(BF)      # the maximum grows from tile to tile
        _batched(q.abs(), rising, v, scale=1.0)
        _batched(q.abs(), rising.flip(1), v, scale=1.0)
        low = torch.finfo(HF).min
        qh, kh = q.to(HF) * 0 + 1, (k.to(HF) * 0).fill_(low / 64)                                  # scores of the type's lowest value
        _batched(qh, kh, v.to(HF), scale=1.0)
    # a NaN or an infinity in a query stays in its row
    q[0, 5, 1] = math.nan
    q[0, 150, 0, 3] = math.inf
    got, clean = ops.attention(q, k, v), ops.attention(q.nan_to_num(0, 0, 0), k, v)
    bad = torch.zeros(tq, 2, dtype=torch.bool, device=DEV)
    bad[5, 1] = bad[150, 0] = True
    assert torch.isnan(got[0, 5, 1]).all() and torch.isnan(got[0, 150, 0]).all() and torch.equal(got[0][~bad], clean[0][~bad])
    # a NaN in a key that counts reaches every row that sees it, in the pass with the polynomial too
    for at in (0, 11, 22, 299):
        kk = k.clone()
        kk[0, at, 0, 0] = math.nan
        assert torch.isnan(ops.attention(q.nan_to_num(0, 0, 0), kk, v)[0, :, 0]).all()


@pytest.mark.parametrize("tq,tk,hq,hkv", [(1, 3000, 8, 2), (20, 6000, 2, 2), (400, 400, 4, 4)], ids=str)
def test_streams_graphs_and_repetition(native_lib, tq, tk, hq, hkv):
    g = _gen(8)
    sets = [(_rand(g, 2, tq, hq, 64), _rand(g, 2, tk, hkv, 64), _rand(g, 2, tk, hkv, 64)) for _ in range(3)]
    lens = torch.tensor([tk, tk // 2], dtype=torch.int32, device=DEV)
    want = [ops.attention(*s, kv_lens=lens) for s in sets]
    torch.cuda.synchronize()
    graphs = []
    for q, k, v in sets[:2]:                                     # two graphs with scratch of their own, replayed at the same time
        ins = [t.clone() for t in (q, k, v)]
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = ops.attention(*ins, kv_lens=lens)
        graphs.append((gr, ins, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(4):
        for (gr, ins, out), st, i in zip(graphs, streams, (0, 1)):
            with torch.cuda.stream(st):
                for t, s in zip(ins, sets[(i + rep) % 3]):
                    t.copy_(s)
                gr.replay()
        torch.cuda.synchronize()
        for (gr, ins, out), i in zip(graphs, (0, 1)):
            assert torch.equal(out, want[(i + rep) % 3])
    lens.copy_(torch.tensor([tk // 3, 1], dtype=torch.int32))    # the replayed graph reads the lengths of now
    graphs[0][0].replay()
    assert torch.equal(graphs[0][2], ops.attention(*graphs[0][1], kv_lens=lens))
    with torch.cuda.stream(streams[0]):                          # eagerly on another stream, several in a row
        outs = [ops.attention(*s) for s in sets]
    torch.cuda.synchronize()
    for o, s in zip(outs, sets):
        assert torch.equal(o, ops.attention(*s))


def test_offsets_past_32_bits(native_lib):
    """The last sequence of a cache of 2.7e9 elements; only its first keys are looked at."""
    g = _gen(9)
    k = torch.empty(10, 65536, 32, 128, dtype=BF, device=DEV)
    v = torch.empty_like(k)
    q = _rand(g, 10, 1, 32, 128)
    lens = [0] * 9 + [300]
    k[9, :300], v[9, :300] = _rand(g, 300, 32, 128), _rand(g, 300, 32, 128)
    _batched(q, k, v, True, kv_lens=lens)
    big = k.view(-1, 32, 128)                                    # and as one packed tensor, from a token behind 2^31 elements on
    off = torch.tensor([9 * 65536, 9 * 65536 + 300], dtype=torch.int32, device=DEV)
    qp = _rand(g, 300, 32, 128)
    out = ops.attention(qp, big, v.view(-1, 32, 128), causal=True, q_offsets=torch.tensor([0, 300], dtype=torch.int32, device=DEV), kv_offsets=off)
    _check(out, None, _reference(qp, k[9, :300], v[9, :300], True, 128 ** -0.5))


def test_nothing_to_do(native_lib):
    z = lambda *s: torch.zeros(*s, dtype=BF, device=DEV)  # noqa: E731
    assert ops.attention(z(0, 5, 2, 64), z(0, 7, 2, 64), z(0, 7, 2, 64)).shape == (0, 5, 2, 64)
    assert ops.attention(z(2, 0, 2, 64), z(2, 7, 2, 64), z(2, 7, 2, 64)).shape == (2, 0, 2, 64)
    for tq in (1, 300):
        out, lse = ops.attention(z(2, tq, 2, 64) + 1, z(2, 0, 2, 64), z(2, 0, 2, 64), return_lse=True)
        assert not out.any() and (lse == -math.inf).all()
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert not ops.attention(z(4, 2, 64) + 1, z(4, 2, 64), z(4, 2, 64), q_offsets=none).any()


def test_refusals(native_lib):
    x = torch.zeros(2, 8, 4, 64, dtype=BF, device=DEV)
    p, off = x.view(16, 4, 64), torch.tensor([0, 16], dtype=torch.int32, device=DEV)
    bad = [
        (TypeError, lambda: ops.attention(x.float(), x.float(), x.float())), (TypeError, lambda: ops.attention(x, x.half(), x)),
        (ValueError, lambda: ops.attention(x, x[:1], x[:1])), (ValueError, lambda: ops.attention(x, x, x[:, :4])),
        (ValueError, lambda: ops.attention(x, x[:, :, :3], x[:, :, :3])), (ValueError, lambda: ops.attention(x[..., :60], x[..., :60], x[..., :60])),
        (ValueError, lambda: ops.attention(*[torch.zeros(1, 8, 1, 136, dtype=BF, device=DEV)] * 3)), (ValueError, lambda: ops.attention(x, x, x, scale=0.0)),
        (ValueError, lambda: ops.attention(x, x, x, scale=-1.0)), (ValueError, lambda: ops.attention(x, x, x, scale=math.nan)),
        (ValueError, lambda: ops.attention(x, x, x, q_offsets=off)), (ValueError, lambda: ops.attention(p, p, p)),
        (ValueError, lambda: ops.attention(x, x, x, kv_offsets=off)), (ValueError, lambda: ops.attention(p, p, p, q_offsets=off, kv_lens=off)),
        (ValueError, lambda: ops.attention(p, p, p, q_offsets=off.long())), (ValueError, lambda: ops.attention(p, p, p, q_offsets=off.cpu())),
        (ValueError, lambda: ops.attention(p, p, p, q_offsets=off, kv_offsets=off[:1])), (ValueError, lambda: ops.attention(x, x, x, kv_lens=off[:1])),
        (ValueError, lambda: ops.attention(x, x, x, out=torch.zeros(2, 8, 4, 64, device=DEV))), (ValueError, lambda: ops.attention(x, x, x, out=x[:1])),
        (ValueError, lambda: ops.attention(x, x, x, out=torch.zeros(2, 8, 64, 4, dtype=BF, device=DEV).transpose(2, 3))),
        (RuntimeError, lambda: ops.attention(x, x.cpu(), x)), (RuntimeError, lambda: ops.attention(x.clone().requires_grad_(), x, x)),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f"call {i} was not refused")
    with torch.no_grad():
        ops.attention(x.clone().requires_grad_(), x, x)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tq,d", [(256, 64), (256, 128), (300, 40), (4, 64)])
def test_hidden_values_weigh_nothing(native_lib, dtype, tq, d):
    """Keys that causality hides have weight 0 exactly, whatever finite value they carry (2^-126 times the largest bf16 is 4)."""
    g = torch.Generator(device="cuda").manual_seed(tq + d)
    q, k, v = (torch.randn(1, tq, 2, d, generator=g, device="cuda").to(dtype) for _ in range(3))
    half = tq // 2
    big = v.clone()
    big[:, half:] = torch.finfo(dtype).max
    clean, hidden = ops.attention(q, k, v, causal=True), ops.attention(q, k, big, causal=True)
    assert torch.equal(clean[:, :half], hidden[:, :half])
