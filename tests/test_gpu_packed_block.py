"""The packed requests' operators run together, as a block's cross attention uses them: every
request's own adapter beside the shared projections, its positions, its own states, and the residual's
norm as the operand of an fp8 linear."""

import pytest
import test_gpu_lora as lora
import test_gpu_packed_attention as attention
import test_gpu_packed_rows as rows_of
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
AXES, DIM, EPS = (44, 42, 42), 128, 1e-6


def inputs(gpu, rows, states, h, hk, requests, seed=0):
    """A block over `rows` rows of width h * 128 and `states` encoder states of width 512."""
    n = h * DIM
    g = torch.Generator(device=gpu).manual_seed(seed + 100)
    return dict(
        q=lora.case(gpu, rows, n, n, 3, 16, seed=seed),
        kv=lora.case(gpu, states, 512, 2 * hk * DIM, 3, 8, seed=seed + 1),
        o=lora.case(gpu, 1, n, n, 3, 16, seed=seed + 2), h=h, hk=hk,
        norm=(1 + 0.2 * torch.randn(n, generator=g, device=gpu)).to(BF16),
        ff=(torch.randn(256, n, generator=g, device=gpu) * n ** -0.5).to(BF16),
        pos=torch.randint(0, 200, (rows, 3), generator=g, device=gpu, dtype=torch.int32),
        qs=torch.zeros(requests + 1, dtype=torch.int32, device=gpu),
        ks=torch.zeros(requests + 1, dtype=torch.int32, device=gpu),
        ids=torch.zeros(requests, dtype=torch.int32, device=gpu))


def fill(b, lengths, keys, ids, gpu):
    b["qs"].copy_(lora.starts(lengths, gpu))
    b["ks"].copy_(lora.starts(keys, gpu))
    b["ids"].copy_(torch.tensor(ids, dtype=torch.int32))


def block(b, w8):
    """Every stage's output."""
    from difflet_amd import kernels
    from difflet_amd.backends.rocm.ops_impl.attention import packed_cross_attention
    from difflet_amd.backends.rocm.ops_impl.embeddings import apply_rotary_axes
    from difflet_amd.backends.rocm.ops_impl.linear import lora_linear
    from difflet_amd.backends.rocm.ops_impl.norm import rms_norm_quantized

    def project(c, x, starts):
        return lora_linear(x, c["w"], c["b"], c["down"], c["up"], c["scale"], starts, b["ids"])

    q = project(b["q"], b["q"]["x"], b["qs"])
    kv = project(b["kv"], b["kv"]["x"], b["ks"])
    k, v = (t.unflatten(-1, (b["hk"], DIM)) for t in kv.chunk(2, dim=-1))
    turned, _ = apply_rotary_axes(q.unflatten(-1, (b["h"], DIM)), None, b["pos"], AXES)
    a = packed_cross_attention(turned, k, v, b["qs"], b["ks"], scale=DIM ** -0.5)
    y = project(b["o"], a.flatten(1), b["qs"])
    codes, scales, hidden = rms_norm_quantized(y, b["norm"], EPS, residual=b["q"]["x"])
    ff = kernels.gemm_call("fp8", codes, w8[0], None, a_scale=scales, w_scale=w8[1])
    return q, kv, turned, a, y, codes, scales, hidden, ff


def check_stages(b, w8, out, lengths, keys, ids):
    """Each stage against 64 bits of what it was given."""
    q, kv, turned, a, y, codes, scales, hidden, ff = out
    lora.check(q, lora.exact(b["q"], lengths, ids))
    lora.check(kv, lora.exact(b["kv"], keys, ids))
    rows_of.check_rope(turned[None], q.unflatten(-1, (b["h"], DIM))[None], b["pos"][None], AXES,
                       10000.0, False, False)
    k, v = (t.unflatten(-1, (b["hk"], DIM)) for t in kv.chunk(2, dim=-1))
    attention.check(a, attention.exact(turned, k, v, lengths, keys, DIM ** -0.5))
    lora.check(y, lora.exact(dict(b["o"], x=a.flatten(1)), lengths, ids))
    h, n = rows_of.norm_exact(y, b["q"]["x"], b["norm"], EPS)
    rows_of.check_codes(n, codes, scales, False)
    assert bool(((hidden.double() - h).abs() <= h.abs() * (2.0 ** -8 + 2.0 ** -23) + 2.0 ** -126).all())
    # codes and scales are exact operands of the linear: fp32 sums and one rounding
    x, w = codes.double() * scales.double()[:, None], w8[0].double() * w8[1].double()[:, None]
    tol = x.abs() @ w.abs().t() * x.shape[1] * 2.0 ** -24 + (x @ w.t()).abs() * (2.0 ** -8 + 2.0 ** -20)
    assert bool(((ff.double() - x @ w.t()).abs() <= tol + 1e-30).all())


CASES = [
    # single tokens, images of requests (one without states, one without rows), rows of no request
    (8, 4, 4, [[1] * 8, [5, 900, 0, 64, 77, 1, 300, 2], [2, 0, -1, 1, 1, 0, 2, 2]]),
    (1500, 8, 8, [[700, 0, 513, 287], [77, 9, 0, 333], [1, 0, 2, -1]]),
    (9000, 16, 16, [[8001, 900], [130, 64], [0, 1]]),
]


@pytest.mark.parametrize("rows,h,hk,what", CASES)
def test_packed_block_stage_by_stage_eager_and_replayed(gpu, rows, h, hk, what):
    from difflet_amd import kernels

    lengths, keys, ids = what
    b = inputs(gpu, rows, sum(keys), h, hk, len(lengths))
    w8 = kernels.quantize_fp8_rowwise(b["ff"])
    fill(b, lengths, keys, ids, gpu)
    check_stages(b, w8, block(b, w8), lengths, keys, ids)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(b, w8)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(b, w8)
    for i in range(3):  # new rows, adapters and cuts
        new = inputs(gpu, rows, sum(keys), h, hk, len(lengths), seed=7 * i + 5)
        b["q"]["x"].copy_(new["q"]["x"])
        b["kv"]["x"].copy_(new["kv"]["x"])
        b["pos"].copy_(new["pos"])
        l2, k2, i2 = (t[i:] + t[:i] for t in (lengths, keys, ids))
        fill(b, l2, k2, i2, gpu)
        graph.replay()
        want = block(b, w8)
        torch.cuda.synchronize()
        for got, w in zip(out, want):
            assert torch.equal(got.view(torch.uint8), w.view(torch.uint8))
        check_stages(b, w8, out, l2, k2, i2)


def test_packed_block_on_two_streams_at_once(gpu):
    """Two batches in flight on streams of their own: each as alone."""
    from difflet_amd import kernels

    batches = []
    for rows, h, hk, (lengths, keys, ids) in CASES:
        b = inputs(gpu, rows, sum(keys), h, hk, len(lengths), seed=rows)
        fill(b, lengths, keys, ids, gpu)
        batches.append((b, kernels.quantize_fp8_rowwise(b["ff"])))
    alone = [block(*b) for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    for _ in range(4):
        out = []
        for s, b in zip(streams, batches):
            with torch.cuda.stream(s):
                out.append(block(*b))
        torch.cuda.synchronize()
        for got, want in zip(out, alone):
            for a, w in zip(got, want):
                assert torch.equal(a.view(torch.uint8), w.view(torch.uint8))
