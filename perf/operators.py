"""What the operators around the quantised linears of a denoise or decode step compute, and at which sizes they are timed.

Three operators:

* `attention`: softmax(scale * q k^T) v of whole sequences, of packed sequences of different lengths (causal or not, heads in
  groups that share keys and values), and of single tokens against a long cache;
* `rotary`: rotary positions with several axes (time, height, width) on the heads of q and k, optionally behind the RMS
  normalisation of each head;
* `gemv_w4`: a few rows of int8 activations times int4 weights with a scale for each group of the inner dimension.

With `own` false `run` computes them from elementary torch operations in fp32 (angles in fp64); with `own` true it makes the
calls of `segquant_b200.ops`.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # joint attention of one block of the denoise step: 4096 image + 333 text tokens, two samples, q | k | v side by side
        # in one projection buffer
        dict(name="attention_joint", op="attention", form="batched", dtype="bf16", batch=2, tq=4429, tk=4429, hq=24, hkv=24,
             d=64, causal=False, joint=True),
        # a text encoder's prompts of very different lengths, packed without padding, four query heads to a key head
        dict(name="attention_packed_causal", op="attention", form="packed", dtype="fp16", lens="517 1 2048 333 77 1023 130 4096 0 255",
             extra="0 0 0 0 0 0 0 0 0 0", hq=32, hkv=8, d=128, causal=True),
        # one long prompt
        dict(name="attention_long_causal", op="attention", form="packed", dtype="bf16", lens="12288", extra="0", hq=16, hkv=2, d=128, causal=True),
        # the next tokens of three prompts behind what their caches hold already (chunked prompts), odd head width
        dict(name="attention_chunk", op="attention", form="packed", dtype="bf16", lens="64 200 7", extra="1000 3100 77", hq=10, hkv=2, d=80, causal=True),
        # one new token of one sequence
        dict(name="attention_token", op="attention", form="cache", dtype="bf16", batch=1, tk=2048, longest=1531, hq=24, hkv=8, d=64, causal=True),
        # one new token each of a serving batch, caches of different fill
        dict(name="attention_tokens", op="attention", form="cache", dtype="fp16", batch=32, tk=16384, longest=16001, hq=32, hkv=8, d=128, causal=True),
        # image tokens of two samples on a 64 x 64 grid, behind the text's tokens on the time axis alone
        dict(name="rotary_image", op="rotary", dtype="bf16", batch=2, grid="1 64 64", text=333, hq=24, hkv=24, d=64, axes="16 24 24",
             pairing="adjacent", norm=True, theta=10000.0),
        # a clip's tokens: 21 frames of 30 x 52 patches
        dict(name="rotary_video", op="rotary", dtype="fp16", batch=1, grid="21 30 52", text=0, hq=16, hkv=16, d=128, axes="44 42 42",
             pairing="adjacent", norm=False, theta=10000.0),
        # one token far along the time axis
        dict(name="rotary_token", op="rotary", dtype="bf16", batch=1, grid="1 1 1", text=0, hq=32, hkv=8, d=128, axes="128",
             pairing="halves", norm=True, theta=500000.0),
        # the modulation of a block: one conditioning vector per sample to six chunks of the hidden size
        dict(name="gemv_modulation", op="gemv_w4", m=2, n=9216, k=1536, group=128, per_token=False, dual=True, dtype="bf16"),
        # a small projection of one row
        dict(name="gemv_small", op="gemv_w4", m=1, n=520, k=512, group=64, per_token=True, dual=False, dtype="fp32"),
        # the widest projection, four rows
        dict(name="gemv_wide", op="gemv_w4", m=4, n=16384, k=12288, group=128, per_token=True, dual=False, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "rotary", "gemv_w4"])
    if op == "attention":
        hkv = rng.choice([1, 2, 3, 8])
        hq = hkv * rng.choice([1, 1, 2, 3, 4, 7, 8])
        d = rng.choice([32, 64, 64, 72, 80, 96, 128, 128])
        form = rng.choice(["batched", "packed", "cache"])
        c = dict(op=op, form=form, dtype=rng.choice(["bf16", "fp16"]), hq=hq, hkv=hkv, d=d)
        if form == "batched":
            t = _log(rng, 1, 4000)
            c.update(batch=rng.choice([1, 2, 3]), tq=t, tk=t if rng.random() < 0.5 else _log(rng, 1, 4000), causal=rng.random() < 0.3, joint=False)
            if c["causal"]:
                c["tk"] = c["tq"]
        elif form == "packed":
            n = rng.choice([1, 2, 5, 9])
            c.update(lens=" ".join(str(_log(rng, 1, 3000)) for _ in range(n)), causal=rng.random() < 0.8,
                     extra=" ".join(str(rng.choice([0, 0, _log(rng, 1, 3000)])) for _ in range(n)))
        else:
            tk = _log(rng, 64, 16000)
            c.update(batch=rng.choice([1, 2, 7, 16]), tk=tk, longest=max(1, int(tk * rng.uniform(0.3, 1.0))), causal=True)
        return c
    if op == "rotary":
        d, axes, pairing = rng.choice([(64, "16 24 24", "adjacent"), (128, "16 56 56", "adjacent"), (128, "44 42 42", "adjacent"), (96, "96", "halves"),
                                       (128, "32 48 48", "halves"), (72, "24 24 24", "adjacent"), (128, "64", "halves"), (64, "20 22 22", "halves")])
        grid = "%d %d %d" % (rng.choice([1, 1, 3, 9]), _log(rng, 1, 50), _log(rng, 1, 50))
        hkv = rng.choice([1, 2, 8, 12])
        return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), batch=rng.choice([1, 2, 3]), grid=grid, text=rng.choice([0, 0, 77, 333]), hq=hkv * rng.choice([1, 3]),
                    hkv=hkv, d=d, axes=axes, pairing=pairing, norm=rng.random() < 0.5, theta=rng.choice([10000.0, 500000.0]))
    group = rng.choice([0, 32, 64, 128, 128, 256])
    k = max(group, 32) * _log(rng, 1, 12288 // max(group, 32))
    return dict(op=op, m=rng.choice([1, 1, 2, 3, 4]), n=_log(rng, 40, 16000), k=k, group=group, per_token=rng.random() < 0.5, dual=rng.random() < 0.3,
                dtype=rng.choice(["bf16", "fp16", "fp32"]))


def _ints(text):
    return [int(v) for v in text.split()]


def _cache_lens(case):
    """Fill of each sequence's cache: the first the longest, the others spread below it."""
    b, top = case["batch"], case["longest"]
    return [max(1, top - (i * 977 * top // 16001) % top) for i in range(b)]


def _pairs(tq, tk, causal):
    """Number of (query, key) pairs that count: query i sees the keys up to i + tk - tq where causal."""
    if not causal:
        return tq * tk
    lo = tk - tq                      # keys that the first query sees, less one
    return sum(max(0, min(tk, i + lo + 1)) for i in range(tq))


def _seqs(case):
    """[(tq, tk)] of an attention case."""
    if case["form"] == "batched":
        return [(case["tq"], case["tk"])] * case["batch"]
    if case["form"] == "cache":
        return [(1, n) for n in _cache_lens(case)]
    return [(n, n + e) for n, e in zip(_ints(case["lens"]), _ints(case["extra"]))]


def _tokens(case):
    return case["text"] + math.prod(_ints(case["grid"]))


def work(case):
    if case["op"] == "attention":
        seqs, d = _seqs(case), case["d"]
        tq, tk = sum(s[0] for s in seqs), sum(s[1] for s in seqs)
        pairs = sum(_pairs(a, b, case["causal"]) for a, b in seqs)
        return {"bytes": 2 * d * (2 * tq * case["hq"] + 2 * tk * case["hkv"]), "flops": 4 * d * case["hq"] * pairs}
    if case["op"] == "rotary":
        es = 4 if case["dtype"] == "fp32" else 2
        rows = case["batch"] * _tokens(case) * (case["hq"] + case["hkv"])
        return {"bytes": 2 * rows * case["d"] * es + 4 * len(_ints(case["axes"])) * _tokens(case),
                "flops": rows * case["d"] * (6 if case["norm"] else 3)}
    m, n, k = case["m"], case["n"], case["k"]
    es, sides = 4 if case["dtype"] == "fp32" else 2, 2 if case["dual"] else 1
    groups = k // case["group"] if case["group"] else 1
    return {"bytes": n * k // 2 + 4 * n * groups + m * k * sides + m * n * es, "flops": 2 * m * n * k * sides}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["op"] == "attention":
        return _prepare_attention(case, randn)
    if case["op"] == "rotary":
        dt, d = _DT[case["dtype"]], case["d"]
        axes, t = _ints(case["axes"]), _tokens(case)
        shift = int(torch.randint(0, 100000 if t == 1 else 8, (1,), generator=gen, device="cuda"))
        f, h, w = _ints(case["grid"])
        idx = torch.arange(f * h * w, device="cuda")
        grid = torch.stack([idx // (h * w) + case["text"] + shift, idx // w % h, idx % w], dim=1)
        text = torch.arange(case["text"], device="cuda")[:, None] * torch.tensor([1, 0, 0], device="cuda")
        pos = torch.cat([text, grid])[:, :len(axes)].to(torch.int32).contiguous()
        st = dict(case=case, q=(1.5 * randn(case["batch"], t, case["hq"], d)).to(dt), k=(1.5 * randn(case["batch"], t, case["hkv"], d)).to(dt),
                  positions=pos, axes=axes, norm_q=None, norm_k=None)
        if case["norm"]:
            st["norm_q"], st["norm_k"] = ((1.0 + 0.2 * randn(d)).to(dt) for _ in range(2))
        return st
    m, n, k, group = case["m"], case["n"], case["k"], case["group"]
    st = dict(case=case, bounds=[0, k])
    st["wq"] = torch.randint(0, 256, (1, n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)

    def codes():
        return (32.0 * randn(1, m, k)).round().clamp(-128, 127)

    x = codes()
    rows = m if case["per_token"] else 1
    st["sx"] = 20.0 + 20.0 * torch.rand(rows, generator=gen, device="cuda")
    st["xq_neg"] = st["sx_neg"] = None
    if case["dual"]:                          # non-negative and negative values in planes of their own
        st["xq_neg"] = x.clamp(max=0).to(torch.int8).view(torch.uint8)
        st["sx_neg"] = 200.0 + 200.0 * torch.rand(rows, generator=gen, device="cuda")
        x = x.clamp(min=0)
    st["xq"] = x.to(torch.int8).view(torch.uint8)
    groups = k // group if group else 1
    st["sw"] = 50.0 + 100.0 * torch.rand(groups, n, generator=gen, device="cuda")       # group-major
    st["bias"] = 0.1 * randn(n)
    return st


def _prepare_attention(case, randn):
    dt, d, hq, hkv = _DT[case["dtype"]], case["d"], case["hq"], case["hkv"]
    st = dict(case=case, seqs=_seqs(case))
    if case["form"] == "packed":
        q_off, kv_off = [0], [0]
        for a, b in st["seqs"]:
            q_off.append(q_off[-1] + a)
            kv_off.append(kv_off[-1] + b)
        st["q"], st["k"], st["v"] = randn(q_off[-1], hq, d).mul_(1.5).to(dt), randn(kv_off[-1], hkv, d).to(dt), randn(kv_off[-1], hkv, d).to(dt)
        st["q_off"], st["kv_off"] = q_off, kv_off
        st["q_offsets"] = torch.tensor(q_off, dtype=torch.int32, device="cuda")
        st["kv_offsets"] = torch.tensor(kv_off, dtype=torch.int32, device="cuda")
    elif case["form"] == "cache":
        b = case["batch"]
        st["q"] = randn(b, 1, hq, d).mul_(1.5).to(dt)
        st["k"], st["v"] = (torch.cat([randn(1, case["tk"], hkv, d).to(dt) for _ in range(b)]) for _ in range(2))
        st["kv_lens"] = torch.tensor([s[1] for s in st["seqs"]], dtype=torch.int32, device="cuda")
    else:
        b, tq, tk = case["batch"], case["tq"], case["tk"]
        if case["joint"]:
            qkv = randn(b, tq, 3, hq, d)
            qkv[:, :, 0] *= 1.5
            qkv = qkv.to(dt)
            st["q"], st["k"], st["v"] = qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]
        else:
            st["q"], st["k"], st["v"] = randn(b, tq, hq, d).mul_(1.5).to(dt), randn(b, tk, hkv, d).to(dt), randn(b, tk, hkv, d).to(dt)
    return st


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if case["op"] == "attention":
        return _run_attention(state, case)
    if case["op"] == "rotary":
        if own:
            from segquant_b200 import ops
            return ops.rotary(state["q"], state["k"], state["positions"], state["axes"], theta=case["theta"], pairing=case["pairing"],
                              norm_q=state["norm_q"], norm_k=state["norm_k"])
        cos, sin = _angles(state["positions"], state["axes"], case["theta"])
        return tuple(_rotate(state[x], cos, sin, state["axes"], case["pairing"], state["norm_" + x]) for x in ("q", "k"))
    if own:
        from segquant_b200 import _lib, ops
        return ops.gemm(_lib.SQ_GEMM_W4A8, state["xq"], state["wq"], case["n"], state["bounds"], state["sx"], state["sw"], xq_neg=state["xq_neg"],
                        sx_neg=state["sx_neg"], per_token=case["per_token"], group_size=case["group"], sw_strides=(0, 0, case["n"], 1),
                        bias=state["bias"], out_dtype=_DT[case["dtype"]])
    return _plain_gemv(state, case)


def _run_attention(st, case):
    if own:
        from segquant_b200 import ops
        kw = dict(causal=case["causal"])
        if case["form"] == "packed":
            kw.update(q_offsets=st["q_offsets"], kv_offsets=st["kv_offsets"])
        elif case["form"] == "cache":
            kw.update(kv_lens=st["kv_lens"])
        return ops.attention(st["q"], st["k"], st["v"], **kw)
    out = torch.empty_like(st["q"], memory_format=torch.contiguous_format)
    for i, (tq, tk) in enumerate(st["seqs"]):
        if tq == 0:
            continue
        if case["form"] == "packed":
            qs, ks = slice(st["q_off"][i], st["q_off"][i] + tq), slice(st["kv_off"][i], st["kv_off"][i] + tk)
            q, k, v, o = st["q"][qs], st["k"][ks], st["v"][ks], out[qs]
        else:
            q, k, v, o = st["q"][i], st["k"][i, :tk], st["v"][i, :tk], out[i]
        o.copy_(_plain_attention(q, k, v, case["causal"]))
    return out


def _plain_attention(q, k, v, causal):
    """q (tq, hq, d), k and v (tk, hkv, d) -> (tq, hq, d) in fp32; a key head at a time, its query heads together."""
    tq, hq, d = q.shape
    tk, hkv, _ = k.shape
    g = hq // hkv
    q, k, v = (t.float().transpose(0, 1) for t in (q, k, v))                      # heads first
    parts = []
    step = max(1, int(2 ** 30 // max(1, g * tq * tk)))                            # key heads at a time: bounded scores
    for h in range(0, hkv, step):
        n = min(step, hkv - h)
        qh = q[h * g:(h + n) * g].reshape(n, g * tq, d)
        s = torch.matmul(qh, k[h:h + n].transpose(1, 2)).view(n, g, tq, tk) * (1.0 / math.sqrt(d))
        if causal:
            i = torch.arange(tq, device=q.device)[:, None] + (tk - tq)
            s = s.masked_fill(torch.arange(tk, device=q.device)[None, :] > i, -math.inf)
        p = torch.exp(s - s.amax(dim=-1, keepdim=True))
        p = p / p.sum(dim=-1, keepdim=True)
        parts.append(torch.matmul(p.view(n, g * tq, tk), v[h:h + n]).view(n * g, tq, d))
    return torch.cat(parts).transpose(0, 1)


def _angles(positions, axes, theta):
    """cos and sin (tokens, rotated pairs): axis a's pair i turns by position * theta^(-2 i / width of the axis)."""
    cols = []
    for a, width in enumerate(axes):
        freq = theta ** (-torch.arange(0, width, 2, dtype=torch.float64, device=positions.device) / width)
        cols.append(positions[:, a].double()[:, None] * freq[None, :])
    ang = torch.cat(cols, dim=1)
    return ang.cos().float(), ang.sin().float()


def _rotate(x, cos, sin, axes, pairing, weight, eps=1e-6):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(dim=-1, keepdim=True) + eps) * weight.float()
    out, at, pair = y.clone(), 0, 0
    for width in axes:
        h = width // 2
        c, s = cos[:, None, pair:pair + h], sin[:, None, pair:pair + h]           # (tokens, 1, pairs)
        if pairing == "adjacent":
            a, b = y[..., at:at + width:2], y[..., at + 1:at + width:2]
            out[..., at:at + width:2], out[..., at + 1:at + width:2] = a * c - b * s, a * s + b * c
        else:
            a, b = y[..., at:at + h], y[..., at + h:at + width]
            out[..., at:at + h], out[..., at + h:at + width] = a * c - b * s, a * s + b * c
        at, pair = at + width, pair + h
    return out.to(x.dtype)


def _plain_gemv(st, case):
    m, n, k, group = case["m"], case["n"], case["k"], case["group"]
    g = k // group if group else 1
    b = st["wq"][0].to(torch.int32)
    w = torch.stack([((b & 15) ^ 8) - 8, ((b >> 4) ^ 8) - 8], dim=-1).float().view(n, g, k // g)      # low nibble first
    y = torch.zeros(m, n, device=w.device)
    for codes, sx in (("xq", "sx"), ("xq_neg", "sx_neg")):
        if st[codes] is None:
            continue
        x = st[codes][0].view(torch.int8).float().view(m, g, k // g)
        acc = torch.matmul(x.transpose(0, 1), w.permute(1, 2, 0))                 # (groups, m, n)
        y += (acc / (st[sx].view(1, -1, 1) * st["sw"][:, None, :])).sum(dim=0)
    return (y + st["bias"]).to(_DT[case["dtype"]])[None]


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(st, case)
    if case["op"] == "rotary":
        return tuple(_exact_rotary(st, case, x) for x in ("q", "k"))
    m, n, k = case["m"], case["n"], case["k"]
    size = case["group"] or k
    byte = st["wq"][0].long()
    y = st["bias"].double().repeat(m, 1)
    for first in range(0, k, size):
        part = byte[:, first // 2:(first + size) // 2]
        low, high = part % 16, part // 16
        low, high = low - 16 * (low > 7), high - 16 * (high > 7)
        for codes, sx in ((st["xq"], st["sx"]), (st["xq_neg"], st["sx_neg"])):
            if codes is not None:
                x = codes[0, :, first:first + size].view(torch.int8).double()
                dot = x[:, 0::2] @ low.double().T + x[:, 1::2] @ high.double().T
                y += dot / sx.double()[:, None] / st["sw"][first // size].double()[None, :]
    return y[None]


def _exact_attention(st, case):
    d, g = case["d"], case["hq"] // case["hkv"]
    q, k, v = st["q"], st["k"], st["v"]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    for i, (tq, tk) in enumerate(st["seqs"]):
        for h in range(case["hq"]):
            if case["form"] == "packed":
                a, b = st["q_off"][i], st["kv_off"][i]
                qs, ks, vs = q[a:a + tq, h], k[b:b + tk, h // g], v[b:b + tk, h // g]
            else:
                qs, ks, vs = q[i, :, h], k[i, :tk, h // g], v[i, :tk, h // g]
            for r in range(0, tq, 4096):
                s = qs[r:r + 4096].double() @ ks.double().T / math.sqrt(d)
                if case["causal"]:
                    rows = torch.arange(r, r + s.shape[0], device=s.device).view(-1, 1)
                    s = torch.where(torch.arange(tk, device=s.device) - (tk - tq) <= rows, s, -math.inf)
                o = torch.exp(s - torch.logsumexp(s, dim=1, keepdim=True)) @ vs.double()
                if case["form"] == "packed":
                    out[a + r:a + r + s.shape[0], h] = o
                else:
                    out[i, r:r + s.shape[0], h] = o
    return out


def _exact_rotary(st, case, name):
    x, w = st[name].double(), st["norm_" + name]
    if w is not None:
        x = x / torch.sqrt(torch.mean(x ** 2, dim=-1, keepdim=True) + 1e-6) * w.double()
    y, at = x.clone(), 0
    for a, width in enumerate(st["axes"]):
        i = torch.arange(width // 2, device=x.device)
        first, second = (at + 2 * i, at + 2 * i + 1) if case["pairing"] == "adjacent" else (at + i, at + i + width // 2)
        turn = st["positions"][:, a, None].double() * torch.exp(-(2.0 * i.double() / width) * math.log(case["theta"]))
        z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones_like(turn), turn)[:, None, :]
        y[..., first], y[..., second] = z.real, z.imag
        at += width
    return y
