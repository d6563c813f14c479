"""Cross attention over packed requests on the GPU against softmax(q k^T scale) v in 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def starts(lengths, dev, first=0):
    s = [first]
    for n in lengths:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32, device=dev)


def exact(q, k, v, lengths, keys, scale, first_q=0, first_k=0):
    """(out, tolerance) in fp64. A probability is rounded to the inputs' type (half a step of it,
    fp16 also 2^-25 where it is subnormal) while the row's sum is not, a score's fp32 sum of dim
    products is off by 2^-24 dim of their absolute sum (to first order the probability by twice that,
    its maximum's error included) and the result is rounded once."""
    h, hk, d = q.shape[1], k.shape[1], q.shape[2]
    half = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    r, c = first_q, first_k
    for n, m in zip(lengths, keys):
        if n and m:
            a = q[r:r + n].double().transpose(0, 1)
            b, w = (t[c:c + m].double().repeat_interleave(h // hk, dim=1).transpose(0, 1)
                    for t in (k, v))
            p = torch.softmax(a @ b.transpose(1, 2) * scale, dim=-1)
            size = (a.abs() @ b.abs().transpose(1, 2)).amax(-1, keepdim=True) * abs(scale)
            part = p @ w.abs()
            o = p @ w
            t = part * (half + 2.0 ** -23 * (d + 8) * size + 2.0 ** -20) + o.abs() * half
            if q.dtype == F16:
                t = t + m * 2.0 ** -25 * w.abs().amax() + 2.0 ** -25
            out[r:r + n], tol[r:r + n] = o.transpose(0, 1), t.transpose(0, 1)
        r, c = r + n, c + m
    return out, tol


def check(got, want):
    out, tol = want
    bad = ~((got.double() - out).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), bad.numel(),
                                 float((got.double() - out).abs().max()))


def case(gpu, dtype, lengths, keys, h, hk, d, seed=0, tail=0, std=1.0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    q = (torch.randn(sum(lengths) + tail, h, d, generator=g, device=gpu) * std).to(dtype)
    k = torch.randn(max(sum(keys), 0), hk, d, generator=g, device=gpu).to(dtype)
    v = torch.randn(max(sum(keys), 0), hk, d, generator=g, device=gpu).to(dtype)
    return q, k, v


LENGTHS = [
    ([1], [1]), ([1], [5000]), ([1] * 16, [4096, 1, 77, 8000, 512, 3001, 0, 226, 1500, 64, 2048,
                                          333, 4095, 7000, 128, 900]),
    ([130, 0, 1, 257], [63, 9, 0, 129]), ([127, 128, 129], [64, 65, 512]), ([1000, 31], [1, 700]),
    ([3] * 70, [17] * 70), ([2500, 4, 700], [300, 1025, 77]),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("h,hk,d", [(4, 4, 128), (28, 4, 128), (6, 2, 64), (3, 1, 40), (2, 2, 100)])
@pytest.mark.parametrize("lengths,keys", LENGTHS)
def test_packed_cross_attention_matches_64_bits(gpu, lengths, keys, h, hk, d, dtype):
    from difflet_amd.backends.rocm.ops_impl.attention import packed_cross_attention

    q, k, v = case(gpu, dtype, lengths, keys, h, hk, d, seed=len(lengths) + d)
    got = packed_cross_attention(q, k, v, starts(lengths, gpu), starts(keys, gpu), scale=d ** -0.5)
    assert got.dtype == dtype
    check(got, exact(q, k, v, lengths, keys, d ** -0.5))


@pytest.mark.parametrize("scale", [None, -0.3, 0.0, 2.0])
def test_packed_cross_attention_scales(gpu, scale):
    from difflet_amd.backends.rocm.ops_impl.attention import packed_cross_attention

    for lengths, keys in (([200, 5], [90, 300]), ([2], [1000])):
        q, k, v = case(gpu, BF16, lengths, keys, 4, 2, 64, std=0.5)
        got = packed_cross_attention(q, k, v, starts(lengths, gpu), starts(keys, gpu), scale=scale)
        check(got, exact(q, k, v, lengths, keys, 1.0 if scale is None else scale))


@pytest.mark.parametrize("lengths,keys", [([300, 41], [77, 200]), ([1, 2, 1], [900, 33, 1500])])
def test_packed_cross_attention_strides_and_rows_of_no_request(gpu, lengths, keys):
    """q, k, v as ranges of fused projections, rows before the first request and behind the last:
    they come out zero, in a given output they stay, and what lies behind the states of a request
    (infinities and NaN here) reaches nobody."""
    from difflet_amd import kernels
    from difflet_amd.backends.rocm.ops_impl.attention import packed_cross_attention

    g = torch.Generator(device=gpu).manual_seed(3)
    h, hk, d = 6, 2, 128
    rows, states = sum(lengths) + 12, sum(keys) + 9
    buf = torch.randn(rows, 2 * h * d + 8, generator=g, device=gpu).to(BF16)
    kv = torch.randn(states, 3 * hk * d, generator=g, device=gpu).to(BF16)
    q = buf[:, h * d:2 * h * d].unflatten(-1, (h, d))
    k, v = (kv[:, i * hk * d:(i + 1) * hk * d].unflatten(-1, (hk, d)) for i in (0, 2))
    kv[:4] = float("inf")
    kv[4 + sum(keys):] = float("nan")
    q_starts, k_starts = starts(lengths, gpu, 5), starts(keys, gpu, 4)
    want = exact(q, k, v, lengths, keys, d ** -0.5, 5, 4)
    got = packed_cross_attention(q, k, v, q_starts, k_starts, scale=d ** -0.5)
    check(got, want)
    assert not bool(got[:5].any()) and not bool(got[5 + sum(lengths):].any())
    out = torch.full((rows, h * d + 4), 7.0, dtype=BF16, device=gpu)
    o = out[:, 4:].unflatten(-1, (h, d))
    kernels.packed_attention(q, k, v, q_starts, k_starts, scale=d ** -0.5, out=o)
    check(o[5:5 + sum(lengths)], tuple(t[5:5 + sum(lengths)] for t in want))
    assert bool((out[:5] == 7).all()) and bool((out[5 + sum(lengths):] == 7).all())
    assert bool((out[:, :4] == 7).all())
    # a request alone
    one = packed_cross_attention(q[5:5 + lengths[0]], k[4:4 + keys[0]], v[4:4 + keys[0]],
                                 starts(lengths[:1], gpu), starts(keys[:1], gpu), scale=d ** -0.5)
    check(one, tuple(t[5:5 + lengths[0]] for t in want))


def test_packed_cross_attention_without_states_or_rows(gpu):
    from difflet_amd.backends.rocm.ops_impl.attention import packed_cross_attention

    q, k, v = case(gpu, BF16, [4, 300], [0, 0], 2, 2, 64)
    z = packed_cross_attention(q, k, v, starts([4, 300], gpu), starts([0, 0], gpu), scale=0.1)
    assert z.shape == q.shape and not bool(z.any())
    z = packed_cross_attention(q, q, q, starts([], gpu), starts([], gpu), scale=0.1)
    assert not bool(z.any())
    z = packed_cross_attention(q[:0], q, q, starts([0], gpu), starts([9], gpu), scale=0.1)
    assert z.shape == (0, 2, 64)


def test_packed_cross_attention_extremes(gpu):
    """Scores of +-1e4 before the softmax, a NaN in one request's states and an infinity in another's
    values: each stays in its request."""
    from difflet_amd.backends.rocm.ops_impl.attention import packed_cross_attention

    for lengths in ([40, 30, 35], [1, 2, 1]):
        keys = [500, 600, 700]
        q, k, v = case(gpu, BF16, lengths, keys, 2, 2, 128, std=100.0)
        got = packed_cross_attention(q, k, v, starts(lengths, gpu), starts(keys, gpu), scale=1.0)
        ref = exact(q, k, v, lengths, keys, 1.0)
        # the largest score alone decides where it leads by more than its own error
        r = c = 0
        for n, m in zip(lengths, keys):
            s = q[r:r + n].double().transpose(0, 1) @ k[c:c + m].double().permute(1, 2, 0)
            top = s.topk(2, dim=-1).values
            sure = ((top[..., 0] - top[..., 1]) > 20).transpose(0, 1)[..., None]
            err = (got[r:r + n].double() - ref[0][r:r + n]).abs()
            assert bool((err * sure <= ref[0][r:r + n].abs() * 2.0 ** -6 + 1e-3).all())
            r, c = r + n, c + m
        k[503, 0, 5] = float("nan")
        v[1105, 1, 9] = float("inf")
        got = packed_cross_attention(q, k, v, starts(lengths, gpu), starts(keys, gpu), scale=0.001)
        a, b = lengths[0], lengths[0] + lengths[1]
        assert bool(got[:a].isfinite().all())
        assert bool(got[a:b, 0].isnan().all()) and bool(got[a:b, 1].isfinite().all())
        assert bool((got[b:, 1, 9] == float("inf")).all()) and bool(got[b:, 0].isfinite().all())


def test_packed_cross_attention_long_strides(gpu):
    """States whose rows lie 16 MB apart, past 32 bits within one request."""
    from difflet_amd.backends.rocm.ops_impl.attention import packed_cross_attention

    far = 1 << 23  # elements
    buf = torch.empty(300 * far + 512, dtype=BF16, device=gpu)
    k = buf.as_strided((300, 2, 64), (far, 64, 1))
    v = buf.as_strided((300, 2, 64), (far, 64, 1), 256)
    g = torch.Generator(device=gpu).manual_seed(0)
    k.copy_(torch.randn(300, 2, 64, generator=g, device=gpu))
    v.copy_(torch.randn(300, 2, 64, generator=g, device=gpu))
    q = torch.randn(50, 2, 64, generator=g, device=gpu).to(BF16)
    got = packed_cross_attention(q, k, v, starts([49, 1], gpu), starts([290, 10], gpu), scale=0.1)
    check(got, exact(q, k, v, [49, 1], [290, 10], 0.1))


@pytest.mark.parametrize("rows", [4, 900])
def test_packed_cross_attention_graph_follows_new_lengths(gpu, rows):
    from difflet_amd.backends.rocm.ops_impl.attention import packed_cross_attention

    q, k, v = case(gpu, BF16, [rows], [3000], 4, 2, 128)
    qs, ks = starts([1, rows - 1], gpu), starts([1000, 2000], gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        packed_cross_attention(q, k, v, qs, ks, scale=0.1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = packed_cross_attention(q, k, v, qs, ks, scale=0.1)
    for i, (lengths, keys) in enumerate((([1, rows - 1], [1000, 2000]), ([rows - 1, 1], [3000, 0]),
                                         ([2, rows - 3], [1, 2222]), ([0, rows], [64, 65]))):
        qs.copy_(starts(lengths, gpu))
        ks.copy_(starts(keys, gpu))
        q.copy_(case(gpu, BF16, [rows], [3000], 4, 2, 128, seed=i)[0])
        graph.replay()
        want = packed_cross_attention(q, k, v, qs, ks, scale=0.1)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        check(out, exact(q, k, v, lengths, keys, 0.1))


def test_packed_cross_attention_row_numbers_out_of_order_stay_inside(gpu):
    """Row numbers past the tensors or going back are clamped: no result is promised for them, but
    the rows of requests whose numbers hold come out right."""
    from difflet_amd.backends.rocm.ops_impl.attention import packed_cross_attention

    q, k, v = case(gpu, BF16, [60], [500], 2, 2, 128)
    qs = torch.tensor([0, 20, 40, 10**9], dtype=torch.int32, device=gpu)
    ks = torch.tensor([0, 100, 50, 2**31 - 1], dtype=torch.int32, device=gpu)
    got = packed_cross_attention(q, k, v, qs, ks, scale=0.1)
    check(got[:20], tuple(t[:20] for t in exact(q, k, v, [20], [100], 0.1)))
    assert not bool(got[20:40].any())
    want = exact(q[40:], k[50:], v[50:], [20], [450], 0.1)
    check(got[40:], want)


def test_packed_cross_attention_compiles(gpu):
    from difflet_amd.backends.rocm.ops_impl.attention import packed_cross_attention

    q, k, v = case(gpu, BF16, [70, 3], [20, 90], 4, 2, 64)
    qs, ks = starts([70, 3], gpu), starts([20, 90], gpu)
    f = torch.compile(lambda q, k, v: packed_cross_attention(q * 2, k, v, qs, ks, scale=0.1) + 1,
                      fullgraph=True, backend="aot_eager")
    want = packed_cross_attention(q * 2, k, v, qs, ks, scale=0.1) + 1
    assert torch.equal(f(q, k, v), want)


MANY = [
    ([9000, 7100], [100, 513], 16, 16, 128), ([12000, 1, 0, 300, 4000], [64, 65, 7, 0, 31], 16, 16, 128),
    ([3333], [1200], 70, 10, 128), ([39000, 700, 26001], [32, 96, 0], 2, 2, 64),
    ([4000, 8100], [77, 300], 24, 12, 64), ([131073], [1], 1, 1, 128), ([300] * 62, [29] * 62, 8, 8, 128),
    ([300] * 63, [29] * 63, 8, 8, 128),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths,keys,h,hk,d", MANY)
def test_packed_cross_attention_of_many_rows(gpu, lengths, keys, h, hk, d, dtype):
    """Whole and ragged tiles of 256 rows, one to eight and more tiles of keys, requests without any,
    heads that share keys; more requests than a wavefront has lanes."""
    from difflet_amd.backends.rocm.ops_impl.attention import packed_cross_attention

    q, k, v = case(gpu, dtype, lengths, keys, h, hk, d, seed=1)
    got = packed_cross_attention(q, k, v, starts(lengths, gpu), starts(keys, gpu), scale=d ** -0.5)
    check(got, exact(q, k, v, lengths, keys, d ** -0.5))


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
def test_packed_cross_attention_of_many_rows_scales(gpu, scale):
    from difflet_amd.backends.rocm.ops_impl.attention import packed_cross_attention

    lengths, keys = [9000, 8000], [200, 333]
    q, k, v = case(gpu, BF16, lengths, keys, 16, 8, 64, std=0.5)
    got = packed_cross_attention(q, k, v, starts(lengths, gpu), starts(keys, gpu), scale=scale)
    check(got, exact(q, k, v, lengths, keys, scale))


@pytest.mark.parametrize("offset", [4, 8])  # rows of the output on 8 or 16 bytes
@pytest.mark.parametrize("h,hk", [(16, 16), (12, 4)])
def test_packed_cross_attention_of_many_rows_strides_and_rows_of_no_request(gpu, h, hk, offset):
    from difflet_amd import kernels
    from difflet_amd.backends.rocm.ops_impl.attention import packed_cross_attention

    g = torch.Generator(device=gpu).manual_seed(5)
    d, lengths, keys = 128, [9001, 600, 3000], [130, 0, 450]
    rows, states = sum(lengths) + 12, sum(keys) + 9
    buf = torch.randn(rows, 2 * h * d + 8, generator=g, device=gpu).to(BF16)
    kv = torch.randn(states, 3 * hk * d, generator=g, device=gpu).to(BF16)
    q = buf[:, h * d:2 * h * d].unflatten(-1, (h, d))
    k, v = (kv[:, i * hk * d:(i + 1) * hk * d].unflatten(-1, (hk, d)) for i in (0, 2))
    kv[:4] = float("inf")
    kv[4 + sum(keys):] = float("nan")
    q_starts, k_starts = starts(lengths, gpu, 5), starts(keys, gpu, 4)
    want = exact(q, k, v, lengths, keys, d ** -0.5, 5, 4)
    got = packed_cross_attention(q, k, v, q_starts, k_starts, scale=d ** -0.5)
    check(got, want)
    end = 5 + sum(lengths)
    assert not bool(got[:5].any()) and not bool(got[end:].any())
    out = torch.full((rows, h * d + 8), 7.0, dtype=BF16, device=gpu)
    o = out[:, offset:offset + h * d].unflatten(-1, (h, d))
    kernels.packed_attention(q, k, v, q_starts, k_starts, scale=d ** -0.5, out=o)
    check(o[5:end], tuple(t[5:end] for t in want))
    assert bool((out[:5] == 7).all()) and bool((out[end:] == 7).all())
    assert bool((out[:, :offset] == 7).all()) and bool((out[:, offset + h * d:] == 7).all())


def test_packed_cross_attention_of_many_rows_extremes(gpu):
    """A NaN in one request's states, an infinity in another's values, scores that grow along the keys
    by far more than the first keys' maximum: each stays in its request."""
    from difflet_amd.backends.rocm.ops_impl.attention import packed_cross_attention

    lengths, keys = [9000, 8000, 300, 1100], [500, 600, 700, 900]
    q, k, v = case(gpu, BF16, lengths, keys, 8, 8, 128)
    qs, ks = starts(lengths, gpu), starts(keys, gpu)
    k[500 + 600 + 700:] = k[500 + 600 + 700:] * torch.linspace(0.1, 30, 900, device=gpu).to(BF16)[:, None, None]
    check(packed_cross_attention(q, k, v, qs, ks, scale=0.3), exact(q, k, v, lengths, keys, 0.3))
    k[503, 0, 5] = float("nan")
    v[1105, 1, 9] = float("inf")
    got = packed_cross_attention(q, k, v, qs, ks, scale=0.001)
    a, b, c = 9000, 17000, 17300
    assert bool(got[:a].isfinite().all()) and bool(got[c:].isfinite().all())
    assert bool(got[a:b, 0].isnan().all()) and bool(got[a:b, 1:].isfinite().all())
    assert bool((got[b:c, 1, 9] == float("inf")).all()) and bool(got[b:c, 0].isfinite().all())


def test_packed_cross_attention_of_many_rows_graph_follows_new_lengths(gpu):
    from difflet_amd.backends.rocm.ops_impl.attention import packed_cross_attention

    rows, states = 17000, 1500
    q, k, v = case(gpu, BF16, [rows], [states], 8, 8, 64)
    qs, ks = starts([1, rows - 1], gpu), starts([1000, 500], gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        packed_cross_attention(q, k, v, qs, ks, scale=0.1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = packed_cross_attention(q, k, v, qs, ks, scale=0.1)
    for i, (lengths, keys) in enumerate((([1, rows - 1], [1000, 500]), ([rows - 1, 1], [1500, 0]),
                                         ([9000, 7000], [1, 1300]), ([0, rows], [64, 65]))):
        qs.copy_(starts(lengths, gpu))
        ks.copy_(starts(keys, gpu))
        q.copy_(case(gpu, BF16, [rows], [states], 8, 8, 64, seed=i)[0])
        graph.replay()
        want = packed_cross_attention(q, k, v, qs, ks, scale=0.1)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        check(out, exact(q, k, v, lengths, keys, 0.1))


def test_packed_cross_attention_of_many_rows_past_32_bits(gpu):
    """Rows of q and of the output and states so far apart that their offsets pass 32 bits."""
    from difflet_amd import kernels

    rows, h, d, keys = 17000, 8, 64, [140, 60]
    g = torch.Generator(device=gpu).manual_seed(0)
    q, o = (torch.empty(rows << 18, dtype=BF16, device=gpu).as_strided((rows, h, d), (1 << 18, d, 1))
            for _ in range(2))
    kv = torch.empty((sum(keys) << 23), dtype=BF16, device=gpu)
    k, v = (kv.as_strided((sum(keys), h, d), (1 << 23, d, 1), i * h * d) for i in (0, 1))
    for t in (q, k, v):
        t.copy_(torch.randn(t.shape, generator=g, device=gpu))
    lengths = [9000, 8000]
    kernels.packed_attention(q, k, v, starts(lengths, gpu), starts(keys, gpu), scale=0.1, out=o)
    check(o, exact(q, k, v, lengths, keys, 0.1))


def test_packed_cross_attention_makes_up_no_gradient(gpu):
    from difflet_amd.backends.rocm.ops_impl.attention import packed_cross_attention

    q, k, v = case(gpu, BF16, [70], [20], 2, 2, 64)
    q.requires_grad_()
    with pytest.raises(RuntimeError):
        packed_cross_attention(q, k, v, starts([70], gpu), starts([20], gpu)).sum().backward()
