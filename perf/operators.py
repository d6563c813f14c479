"""Operators over the packed rows of several requests, as they are measured: each in a plain form
(elementary torch operations in 32 bits) and, where `own` is true, through the framework's calls.

A case is a dict of plain values whose "op" is one of

  lora   a linear shared by the requests of a batch beside a low-rank adapter of each request's own
         (ops_impl.linear.lora_linear); weights bf16, per-channel fp8 or MXFP8
  norm   the residual's addition, RMSNorm and an 8-bit output with scales, the A operand of an fp8
         linear (ops_impl.norm.rms_norm_quantized)
  rope   rotary embedding of q and k from positions on several axes
         (ops_impl.embeddings.apply_rotary_axes)
  cross  cross attention of each request's rows to the states of its own encoder, of another length
         (ops_impl.attention.packed_cross_attention)

The rows of a batch's requests lie behind one another in one tensor; "lengths" names their rows,
"keys" their encoder states, both as comma-separated numbers. The widths are those of the
repository's model configurations (FLUX and Qwen-Image: hidden 3072, 24 heads; Wan: 5120, 40 heads;
T5: 4096); grouped key heads are generic.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
BF16 = torch.bfloat16
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
EPS = 1e-6
TINY = 2.0 ** -112  # the per-row fp8 law's smallest row maximum
THETA = 10000.0

# (in, out) of the linears that adapters are trained for, bf16 and quantized
LINEARS = [(3072, 3072), (3072, 9216), (3072, 12288), (12288, 3072), (3072, 18432), (5120, 5120),
           (5120, 13824), (13824, 5120), (4096, 10240)]
MOST_FLOPS = 4.9e12  # a drawn case's matrix work stays below the largest listed linear's
MOST_SCORES = 1.9e9  # and a drawn attention's padded scores below the largest listed one's


def listed():
    return [
        # adaLN modulation of a double block for eight requests' timestep embeddings at once, one
        # row each, an adapter each but for one request: bound by the shared weight
        dict(name="lora_modulation", op="lora", kind="bf16", lengths="1,1,1,1,1,1,1,1",
             adapters="0,1,2,-1,3,4,5,6", tail=0, k=3072, n=18432, rank=16),
        # FLUX's MLP over three requests of 1024 x 1024, 512 x 512 and an odd size
        dict(name="lora_images", op="lora", kind="bf16", lengths="4096,1024,2021",
             adapters="1,0,2", tail=0, k=3072, n=12288, rank=32),
        # the fused q/k/v projection of two requests, text and image rows, per-channel fp8; the
        # last rows pad the batch to its bucket
        dict(name="lora_fp8", op="lora", kind="fp8", lengths="4608,4173", adapters="0,1", tail=179,
             k=3072, n=9216, rank=16),
        # Wan's FFN over the 32760 video tokens of 480p x 81 frames and one of 17 frames, MXFP8
        dict(name="lora_video", op="lora", kind="mx", lengths="32760,1365", adapters="0,1", tail=0,
             k=5120, n=13824, rank=64),
        # one token of a text encoder's width, per-token fp8: latency alone
        dict(name="norm_token", op="norm", dtype="bf16", format="fp8_rowwise", rows=1, dim=4096),
        # the rows of 480p x 81 frames at Wan's width, MXFP8
        dict(name="norm_video", op="norm", dtype="bf16", format="mxfp8", rows=32760, dim=5120),
        # text rows of an odd count with grouped key heads, halves rotated, frequencies shared by
        # the axes, positions past 2^20
        dict(name="rope_text", op="rope", dtype="bf16", batch=1, seq=77, heads=28, kv_heads=4,
             dim=128, axes="32,48,48", layout="halves", shared=True, far=1 << 21, grid=False),
        # q and k of 480p x 81 frames, Wan's axes
        dict(name="rope_video", op="rope", dtype="bf16", batch=1, seq=32760, heads=40, kv_heads=40,
             dim=128, axes="44,42,42", layout="interleaved", shared=False, far=104, grid=True),
        # two batch elements in fp32, FLUX's axes
        dict(name="rope_fp32", op="rope", dtype="fp32", batch=2, seq=1541, heads=24, kv_heads=24,
             dim=128, axes="16,56,56", layout="interleaved", shared=False, far=128, grid=False),
        # single tokens of 16 requests reading states of very different lengths, grouped key heads
        dict(name="cross_tokens", op="cross", dtype="bf16", lengths=",".join(["1"] * 16),
             keys="4096,1,77,8000,512,3001,0,226,1500,64,2048,333,4095,7000,128,900", heads=28,
             kv_heads=4, dim=128),
        # the images of three requests and their prompts, one of them without any
        dict(name="cross_images", op="cross", dtype="bf16", lengths="4096,1024,6889,1600",
             keys="512,77,256,0", heads=24, kv_heads=24, dim=128),
        # Wan's cross attention: 480p x 81 frames of a request and of a shorter clip
        dict(name="cross_video", op="cross", dtype="bf16", lengths="32760,9360", keys="512,226",
             heads=40, kv_heads=40, dim=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(values):
    return ",".join(str(v) for v in values)


def _numbers(text):
    return [int(v) for v in text.split(",")]


def draw(rng):
    op = rng.choice(["lora", "lora", "norm", "rope", "cross", "cross"])
    if op == "lora":
        kind = rng.choice(["bf16", "bf16", "fp8", "mx"])
        k, n = rng.choice(LINEARS)
        rows = _log(rng, 1, min(32760, MOST_FLOPS / (2 * k * n)))
        count = rng.randint(1, min(rows, 24))
        cuts = sorted(rng.randint(0, rows) for _ in range(count - 1))
        lengths = [b - a for a, b in zip([0] + cuts, cuts + [rows])]
        return dict(op=op, kind=kind, lengths=_text(lengths),
                    adapters=_text(rng.randint(-1, 7) for _ in lengths),
                    tail=rng.choice([0, 0, rng.randint(1, 200)]), k=k, n=n,
                    rank=rng.choice([4, 8, 16, 16, 32, 64, 128]))
    if op == "norm":
        fmt = rng.choice(["fp8_rowwise", "mxfp8"])
        dim = 128 * rng.randint(4, 64) if fmt == "mxfp8" else 8 * rng.randint(16, 1024)
        return dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), format=fmt,
                    rows=_log(rng, 1, 1.6e8 / dim), dim=dim)
    if op == "rope":
        dim = rng.choice([64, 96, 128, 128])
        quarter = dim // 8
        axes = rng.choice([(4 * quarter, 2 * quarter, 2 * quarter), (2 * quarter, 6 * quarter),
                           (2 * quarter, 2 * quarter, 2 * quarter), (dim,)])
        kv = rng.choice([4, 8, 24])
        heads = kv * rng.choice([1, 1, 3])
        batch = rng.randint(1, 3)
        return dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), batch=batch,
                    seq=_log(rng, 1, 60000 / batch), heads=heads, kv_heads=kv, dim=dim,
                    axes=_text(axes), layout=rng.choice(["interleaved", "halves"]),
                    shared=rng.random() < 0.5, far=_log(rng, 16, 1 << 21),
                    grid=rng.random() < 0.5)
    count = rng.randint(1, 16)
    kv = rng.choice([4, 8, 24])
    heads = kv * rng.choice([1, 1, 4])
    if rng.random() < 0.4:  # few rows, long states
        lengths = [rng.randint(1, 4) for _ in range(count)]
        keys = [rng.choice([0, _log(rng, 1, 8192), _log(rng, 1, 8192)]) for _ in range(count)]
    else:
        keys = [rng.choice([_log(rng, 1, 1200), _log(rng, 32, 512)]) for _ in range(count)]
        most = max(1, int(MOST_SCORES / (count * heads * max(keys))))
        lengths = [_log(rng, 1, min(most, 33000)) for _ in range(count)]
    if max(keys) == 0:
        keys[0] = 77
    return dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), lengths=_text(lengths),
                keys=_text(keys), heads=heads, kv_heads=kv, dim=rng.choice([64, 128, 128]))


# ------------------------------------------------------------------------------- inputs
def _starts(lengths):
    s = [0]
    for n in lengths:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32, device=DEV)


def _swizzle(k):
    """Position r * 4 + j of a 512-wide tile (or of the remainder) holds its element
    j * (tile / 4) + r: the order in which MXFP8 rows are stored and cut in blocks of 32."""
    full = k // 512 * 512
    i = torch.arange(k, device=DEV)
    parts = [i[:full].view(-1, 4, 128).transpose(1, 2).reshape(-1),
             i[full:].view(4, -1).t().reshape(-1)]
    return torch.cat(parts)


def _e4m3(v):
    """v rounded to e4m3, past its range to its largest."""
    return v.clamp(-448.0, 448.0).to(E4M3)


def _rowwise(x):
    """Codes and scales [rows] of x by the per-row law: scale = max|row| / 448. Both divisions are
    tensor by tensor: torch takes one by a number as a product with its reciprocal."""
    a = x.abs().amax(dim=-1, keepdim=True).clamp_min(TINY)
    top = torch.full_like(a, 448.0)
    return _e4m3(x * (top / a)), (a / top)[..., 0]


def _blocks(x):
    """Codes and E8M0 scales [rows, dim / 32] of x, already in swizzle order, by the block law:
    the exponent of the scale is 7 below that of the block's largest value."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    e = torch.frexp(b.abs().amax(dim=-1))[1].to(torch.int64) - 1 + 127  # biased exponent
    e = torch.where(b.abs().amax(dim=-1) == 0, torch.zeros_like(e), e)
    s = (e - 7).clamp(0, 255)
    codes = _e4m3(b * torch.exp2((127 - s).to(x.dtype))[..., None])
    return codes.reshape(x.shape), s.to(torch.uint8)


def _values(codes, s, kind):
    """What codes and scales stand for, in 32 bits."""
    v = codes.to(torch.float32)
    if kind == "fp8":
        return v * s[:, None]
    return (v.view(v.shape[0], -1, 32) * torch.exp2(s.to(torch.float32) - 127.0)[..., None]
            ).view(v.shape)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 13)

    def randn(*shape, std=1.0, dtype=BF16):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)

    st = {"case": case}
    op = case["op"]
    if op == "lora":
        lengths, ids = _numbers(case["lengths"]), _numbers(case["adapters"])
        rows, k, n, r = sum(lengths) + case["tail"], case["k"], case["n"], case["rank"]
        count = max(max(ids), 0) + 1
        x = randn(rows, k)
        x[:, :: 97] *= 8  # channels that stand out, as activations have
        w = randn(n, k, std=k ** -0.5)
        st.update(x=x, bias=randn(n, std=0.1), down=randn(count, r, k, std=k ** -0.5),
                  up=randn(count, n, r, std=0.5 * r ** -0.5),
                  scale=torch.rand(count, generator=g, device=DEV) + 0.5,
                  starts=_starts(lengths), adapter=torch.tensor(ids, dtype=torch.int32, device=DEV))
        if case["kind"] == "bf16":
            st.update(w=w, w_scale=None)
        elif case["kind"] == "fp8":
            codes, s = _rowwise(w.float())
            st.update(w=codes, w_scale=s)
        else:
            codes, s = _blocks(w.float()[:, _swizzle(k)])
            st.update(w=codes, w_scale=s)
    elif op == "norm":
        dt, rows, dim = DTYPES[case["dtype"]], case["rows"], case["dim"]
        x = randn(rows, dim, dtype=dt)
        x[:, :: 61] *= 16
        st.update(x=x, residual=randn(rows, dim, std=2.0, dtype=dt),
                  weight=(1 + 0.2 * torch.randn(dim, generator=g, device=DEV)).to(dt))
    elif op == "rope":
        dt, b, s = DTYPES[case["dtype"]], case["batch"], case["seq"]
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        buf = randn(b, s, (h + 2 * hk) * d, dtype=dt)  # a fused projection's output
        q, k, _ = buf.split([h * d, hk * d, hk * d], dim=-1)
        axes = _numbers(case["axes"])
        if case["grid"]:
            w = max(1, min(case["far"], int(math.sqrt(s / 21)) or 1))
            i = torch.arange(s, device=DEV)
            pos = torch.stack([i // (w * w), i // w % w, i % w][-len(axes):], dim=-1)
            pos = pos.to(torch.int32).expand(b, s, len(axes)).contiguous()
        else:
            pos = torch.randint(0, case["far"], (b, s, len(axes)), generator=g, device=DEV,
                                dtype=torch.int32)
        st.update(q=q.view(b, s, h, d), k=k.view(b, s, hk, d), positions=pos, axes=tuple(axes))
    else:
        dt, h, hk, d = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
        lengths, keys = _numbers(case["lengths"]), _numbers(case["keys"])
        kv = randn(sum(keys), 2 * hk * d, dtype=dt)  # the states' fused k / v projection
        k, v = kv.split([hk * d, hk * d], dim=-1)
        st.update(q=randn(sum(lengths), h, d, std=1.5, dtype=dt), k=k.view(-1, hk, d),
                  v=v.view(-1, hk, d), q_starts=_starts(lengths), k_starts=_starts(keys),
                  most_q=max(lengths), most_k=max(keys))
    return st


# ------------------------------------------------------------------------------- one pass
def run(st):
    case = st["case"]
    if own:
        return _run_own(st, case)
    return {"lora": _lora, "norm": _norm, "rope": _rope, "cross": _cross}[case["op"]](st, case)


def _run_own(st, case):
    from difflet_amd.backends.rocm.ops_impl import attention, embeddings, linear, norm

    if case["op"] == "lora":
        return linear.lora_linear(st["x"], st["w"], st["bias"], st["down"], st["up"], st["scale"],
                                  st["starts"], st["adapter"], weight_scale=st["w_scale"])
    if case["op"] == "norm":
        codes, scales, hidden = norm.rms_norm_quantized(st["x"], st["weight"], EPS,
                                                        residual=st["residual"],
                                                        format=case["format"])
        return codes, _as_scales(scales), hidden
    if case["op"] == "rope":
        return embeddings.apply_rotary_axes(st["q"], st["k"], st["positions"], st["axes"],
                                            theta=THETA, layout=case["layout"],
                                            shared_frequencies=case["shared"])
    return attention.packed_cross_attention(st["q"], st["k"], st["v"], st["q_starts"],
                                            st["k_starts"], scale=case["dim"] ** -0.5)


def _as_scales(s):
    """E8M0 scales as the powers of two that they stand for."""
    return s.view(torch.float8_e8m0fnu) if s.dtype == torch.uint8 else s


def _row_adapters(starts, adapter, rows):
    """The adapter of each row, -1 for none and for rows behind the last request."""
    row = torch.arange(rows, device=DEV, dtype=torch.int32)
    request = torch.searchsorted(starts[1:], row, right=True)
    ids = torch.cat([adapter, adapter.new_full((1,), -1)])
    return ids[request].to(torch.int64)


def _lora(st, case):
    x = st["x"].float()
    if case["kind"] == "bf16":
        y = x @ st["w"].float().t()
    elif case["kind"] == "fp8":
        y = _values(*_rowwise(x), "fp8") @ _values(st["w"], st["w_scale"], "fp8").t()
    else:
        y = (_values(*_blocks(x[:, _swizzle(case["k"])]), "mx")
             @ _values(st["w"], st["w_scale"], "mx").t())
    y += st["bias"].float()
    down, up = st["down"].float(), st["up"].float()
    count, r, k = down.shape
    ids = _row_adapters(st["starts"], st["adapter"], x.shape[0])
    hot = (ids[:, None] == torch.arange(count, device=DEV)).float() * st["scale"]
    v = (x @ down.reshape(count * r, k).t()).view(-1, count, r) * hot[..., None]
    y += v.view(-1, count * r) @ up.transpose(1, 2).reshape(count * r, -1)
    return y.to(BF16)


def _norm(st, case):
    h = st["x"].float() + st["residual"].float()
    y = h * torch.rsqrt(h.square().mean(dim=-1, keepdim=True) + EPS) * st["weight"].float()
    if case["format"] == "fp8_rowwise":
        codes, s = _rowwise(y)
    else:
        codes, s = _blocks(y[:, _swizzle(case["dim"])])
    return codes, _as_scales(s), h.to(st["x"].dtype)


def _angles(case, positions, axes):
    """cos and sin [batch, seq, pairs], angles in 64 bits."""
    freqs, axis, total = [], [], sum(axes)
    for a, d in enumerate(axes):
        i = torch.arange(0, d, 2, dtype=torch.float64, device=DEV)
        first = 2 * len(axis) if case["shared"] else 0
        freqs.append(THETA ** (-(i + first) / (total if case["shared"] else d)))
        axis += [a] * (d // 2)
    pos = positions.double()[..., torch.tensor(axis, device=DEV)]
    ang = pos * torch.cat(freqs)
    return ang.cos(), ang.sin()


def _rotate(x, cos, sin, layout):
    """x [batch, seq, heads, dim] with its first 2 * pairs channels rotated, in cos's type."""
    pairs = cos.shape[-1]
    cos, sin = cos[:, :, None], sin[:, :, None]
    r = x[..., : 2 * pairs].to(cos.dtype)
    if layout == "interleaved":
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = r[..., :pairs], r[..., pairs:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([y, x[..., 2 * pairs:].to(cos.dtype)], dim=-1)


def _rope(st, case):
    cos, sin = (t.float() for t in _angles(case, st["positions"], st["axes"]))
    return tuple(_rotate(st[n], cos, sin, case["layout"]).to(st[n].dtype) for n in ("q", "k"))


def _padded(t, starts, most):
    """[requests, most, ...] of packed rows, clamped where a request has fewer; and which are."""
    at = starts[:-1, None].long() + torch.arange(most, device=DEV)
    there = at < starts[1:, None]
    return t[at.clamp(max=max(t.shape[0] - 1, 0))], there


def _cross(st, case):
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    q, q_there = _padded(st["q"], st["q_starts"], st["most_q"])
    k, k_there = _padded(st["k"], st["k_starts"], st["most_k"])
    v, _ = _padded(st["v"], st["k_starts"], st["most_k"])
    n, mq, mk = q.shape[0], q.shape[1], k.shape[1]
    # [requests * key heads, rows * group, dim]: the query heads of a key head side by side
    q = q.view(n, mq, hk, h // hk, d).permute(0, 2, 1, 3, 4).float().reshape(n * hk, -1, d)
    k = k.permute(0, 2, 3, 1).float().reshape(n * hk, d, mk).contiguous()
    v = v.permute(0, 2, 1, 3).float().reshape(n * hk, mk, d).contiguous()
    s = torch.bmm(q, k).mul_(d ** -0.5).view(n, hk, -1, mk)
    s.masked_fill_(~k_there[:, None, None], -math.inf)
    top = s.amax(dim=-1, keepdim=True).clamp_min(-3e38)  # a request without states: no row of -inf
    p = s.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    o = torch.bmm(p.view(n * hk, -1, mk), v).view(n, hk, -1, d)
    o = o / torch.where(total == 0, torch.ones_like(total), total)
    o = o.view(n, hk, mq, h // hk, d).permute(0, 2, 1, 3, 4).reshape(n, mq, h, d)
    return o[q_there].to(st["q"].dtype)


# ------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "lora":
        lengths, ids = _numbers(case["lengths"]), _numbers(case["adapters"])
        rows, k, n, r = sum(lengths) + case["tail"], case["k"], case["n"], case["rank"]
        used = len({a for a, m in zip(ids, lengths) if a >= 0 and m > 0})
        adapted = sum(m for a, m in zip(ids, lengths) if a >= 0)
        weight = {"bf16": 2.0, "fp8": 1.0, "mx": 1 + 1 / 32}[case["kind"]] * n * k
        return {"bytes": weight + 2 * n + rows * (k + n) * 2 + used * r * (k + n) * 2,
                "flops": 2.0 * rows * k * n + 2.0 * adapted * r * (k + n)}
    if op == "norm":
        size = 4 if case["dtype"] == "fp32" else 2
        out = 1 + (1 / 32 if case["format"] == "mxfp8" else 4 / case["dim"])
        return {"bytes": case["rows"] * case["dim"] * (3 * size + out) + case["dim"] * size,
                "flops": 6.0 * case["rows"] * case["dim"]}
    if op == "rope":
        size = 4 if case["dtype"] == "fp32" else 2
        rows = case["batch"] * case["seq"]
        heads = case["heads"] + case["kv_heads"]
        return {"bytes": rows * (heads * case["dim"] * 2 * size + 4 * len(_numbers(case["axes"]))),
                "flops": 3.0 * rows * heads * sum(_numbers(case["axes"]))}
    lengths, keys = _numbers(case["lengths"]), _numbers(case["keys"])
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    return {"bytes": 4.0 * sum(lengths) * h * d
            + 4.0 * sum(m for m, q in zip(keys, lengths) if q > 0) * hk * d,
            "flops": 4.0 * h * d * sum(a * b for a, b in zip(lengths, keys))}


# ------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """What run() returns, by each operator's definition in 64 bits, request by request."""
    st = prepare(case, seed)
    if case["op"] == "lora":
        return _exact_lora(st, case)
    if case["op"] == "norm":
        return _exact_norm(st, case)
    if case["op"] == "rope":
        return _exact_rope(st, case)
    return _exact_cross(st, case)


def _exact_codes(x, block):
    """(values, scales) of fp64 x by the 8-bit laws: per row, or in blocks of 32 of the swizzled
    order. The per-row law's reciprocal and products are 32-bit by definition: of bf16 values a
    good part lies on a border between two codes, where the next bits would decide."""
    if not block:
        a = x.abs().amax(dim=-1, keepdim=True).clamp_min(TINY)
        codes = (x * (448 / a).float().double()).float().double().clamp(-448, 448)
        return _nearest_e4m3(codes), (a / 448)[:, 0]
    k = x.shape[-1]
    order = torch.cat([torch.arange(t, min(t + 512, k)).view(4, -1).t().reshape(-1)
                       for t in range(0, k, 512)]).to(DEV)
    b = x[:, order].view(x.shape[0], -1, 32)
    top = b.abs().amax(dim=-1)
    e = torch.floor(torch.log2(top))  # fixed below where the logarithm rounds over a power
    e = torch.where(torch.exp2(e) > top, e - 1, e)
    e = torch.where(torch.exp2(e + 1) <= top, e + 1, e)
    s = torch.exp2((e - 7).clamp_min(-127))
    return _nearest_e4m3((b / s[..., None]).clamp(-448, 448)).view(x.shape), s


def _nearest_e4m3(v):
    """fp64 v in [-448, 448] to the nearest e4m3 value, ties to even: steps of 2^(e - 3), and of
    2^-9 below 2^-6."""
    e = torch.frexp(v)[1].to(torch.float64) - 1
    step = torch.exp2(torch.where(v == 0, torch.full_like(e, -6.0), e).clamp_min(-6) - 3)
    return torch.round(v / step) * step


def _exact_lora(st, case):
    x = st["x"].double()
    if case["kind"] == "bf16":
        y = x @ st["w"].double().t()
    elif case["kind"] == "fp8":
        codes, s = _exact_codes(x, False)
        y = (codes * s[:, None]) @ (st["w"].double() * st["w_scale"].double()[:, None]).t()
    else:
        codes, s = _exact_codes(x, True)
        w = st["w"].double().view(case["n"], -1, 32)
        w = (w * torch.exp2(st["w_scale"].double() - 127)[..., None]).view(case["n"], -1)
        y = (codes.view(x.shape[0], -1, 32) * s[..., None]).view(x.shape) @ w.t()
    y += st["bias"].double()
    row = 0
    for length, a in zip(_numbers(case["lengths"]), _numbers(case["adapters"])):
        if a >= 0 and length > 0:
            low = x[row:row + length] @ st["down"][a].double().t()
            y[row:row + length] += st["scale"][a].double() * (low @ st["up"][a].double().t())
        row += length
    return y


def _exact_norm(st, case):
    h = st["x"].double() + st["residual"].double()
    y = h / torch.sqrt(h.pow(2).mean(dim=-1, keepdim=True) + EPS) * st["weight"].double()
    codes, s = _exact_codes(y, case["format"] == "mxfp8")
    return codes, s, h


def _exact_rope(st, case):
    axes, total = st["axes"], sum(st["axes"])
    pos = st["positions"].cpu().double()
    ang, done = [], 0
    for a, d in enumerate(axes):
        for j in range(d // 2):
            f = THETA ** (-2.0 * (done + j) / total if case["shared"] else -2.0 * j / d)
            ang.append(pos[..., a] * f)
        done += d // 2
    turn = torch.exp(1j * torch.stack(ang, dim=-1)).to(DEV)[:, :, None]
    out = []
    for x in (st["q"].double(), st["k"].double()):
        if case["layout"] == "interleaved":
            z = torch.view_as_complex(x[..., :total].reshape(*x.shape[:-1], -1, 2).contiguous())
            y = torch.view_as_real(z * turn).flatten(-2)
        else:
            z = torch.complex(x[..., : total // 2].contiguous(),
                              x[..., total // 2:total].contiguous()) * turn
            y = torch.cat([z.real, z.imag], dim=-1)
        out.append(torch.cat([y, x[..., total:]], dim=-1))
    return tuple(out)


def _exact_cross(st, case):
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    r, c = 0, 0
    for length, keys in zip(_numbers(case["lengths"]), _numbers(case["keys"])):
        for j in range(h if keys and length else 0):
            q = st["q"][r:r + length, j].double()
            k = st["k"][c:c + keys, j * hk // h].double()
            v = st["v"][c:c + keys, j * hk // h].double()
            out[r:r + length, j] = torch.softmax(q @ k.t() * d ** -0.5, dim=-1) @ v
        r, c = r + length, c + keys
    return out
