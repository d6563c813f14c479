"""Low-rank adapters of packed requests beside a shared linear, on the GPU against 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def starts(lengths, dev, first=0):
    s = [first]
    for n in lengths:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32, device=dev)


def case(gpu, rows, k, n, adapters, rank, seed=0, bias=True):
    g = torch.Generator(device=gpu).manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g, device=gpu) * std).to(BF16)  # noqa: E731
    return dict(x=r(rows, k), w=r(n, k, std=k ** -0.5), b=r(n) if bias else None,
                down=r(adapters, rank, k, std=k ** -0.5), up=r(adapters, n, rank, std=rank ** -0.5),
                scale=torch.rand(adapters, generator=g, device=gpu) + 0.5)


def exact(c, lengths, ids, base=None, first=0, extra=0.0):
    """(y, tolerance) in fp64 (base: x W^T without bias). The products of a bf16 row are summed in
    fp32, off by at most 2^-24 K times their absolute sum, the rank values likewise and rounded to
    bf16 (2^-8 of each), and the result once (2^-8). `extra` times base's own tolerance for fp8."""
    x, w = c["x"].double(), c["w"].double() if base is None else None
    k = x.shape[1]
    y = x @ w.t() if base is None else base.clone()
    size = x.abs() @ c["w"].double().abs().t() if base is None else torch.zeros_like(y)
    tol = size * k * 2.0 ** -24 + extra
    if c["b"] is not None:
        y = y + c["b"].double()
    r = first
    for n, a in zip(lengths, ids):
        if n and 0 <= a < c["down"].shape[0]:
            d, u, s = c["down"][a].double(), c["up"][a].double(), c["scale"][a].double()
            v = x[r:r + n] @ d.t() * s
            vt = v.abs() * (2.0 ** -8 + 2.0 ** -20) + x[r:r + n].abs() @ d.abs().t() * s * k * 2.0 ** -24
            y[r:r + n] += v @ u.t()
            tol[r:r + n] += vt @ u.abs().t() + v.abs() @ u.abs().t() * 2.0 ** -16
        r += n
    return y, tol + y.abs() * 2.0 ** -8 + 1e-30


def check(got, want):
    y, tol = want
    bad = ~((got.double() - y).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), bad.numel(), float((got.double() - y).abs().max()))


def run(c, lengths, ids, gpu, first=0, **kw):
    from difflet_amd.backends.rocm.ops_impl.linear import lora_linear

    return lora_linear(c["x"], kw.pop("weight", c["w"]), c["b"], c["down"], c["up"], c["scale"],
                       starts(lengths, gpu, first),
                       torch.tensor(ids, dtype=torch.int32, device=gpu), **kw)


# rows, K, N: small tiles whole and in K pieces, 256 x 256 tiles whole and on the split schedule
SHAPES = [(1, 128, 64), (1, 3072, 9216), (8, 3072, 3072), (70, 640, 132), (513, 1024, 1028),
          (1100, 3072, 3072), (2500, 512, 2048), (5000, 1024, 3072), (4600, 3072, 4096)]


@pytest.mark.parametrize("rank", [1, 4, 8, 16, 40, 64, 128])
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_lora_linear_matches_64_bits(gpu, rows, k, n, rank):
    c = case(gpu, rows, k, n, 3, rank, seed=rows + rank)
    cut = [rows // 3, 0, rows - rows // 3 - rows // 5, rows // 5]
    for lengths, ids in (([rows], [1]), (cut, [2, 0, -1, 0])):
        check(run(c, lengths, ids, gpu), exact(c, lengths, ids))


@pytest.mark.parametrize("rows,k,n", [(300, 256, 512), (64, 3072, 1024), (2600, 256, 4096)])
def test_lora_linear_many_requests_in_a_tile(gpu, rows, k, n):
    """One row a request, each of 60 adapters in no order: a tile holds more adapters than a stage."""
    c = case(gpu, rows, k, n, 60, 16)
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(-1, 60, (rows,), generator=g).tolist()
    check(run(c, [1] * rows, ids, gpu), exact(c, [1] * rows, ids))
    lengths = torch.randint(0, 3, (rows // 2,), generator=g).tolist()  # rows left over: no request
    check(run(c, lengths, ids[: rows // 2], gpu), exact(c, lengths, ids[: rows // 2]))


def test_lora_linear_more_requests_than_are_kept_in_lds(gpu):
    rows = 2600
    c = case(gpu, rows, 256, 256, 5, 8)
    ids = [i % 6 - 1 for i in range(rows)]
    check(run(c, [1] * rows, ids, gpu), exact(c, [1] * rows, ids))


@pytest.mark.parametrize("rows,k,n", [(37, 100, 70), (300, 72, 33), (9, 64, 6), (1, 36, 1)])
def test_lora_linear_odd_widths(gpu, rows, k, n):
    c = case(gpu, rows, k, n, 2, 5)
    check(run(c, [rows // 2, rows - rows // 2], [1, 0], gpu),
          exact(c, [rows // 2, rows - rows // 2], [1, 0]))


def test_lora_linear_layouts(gpu):
    """A column range of a wider input, a strided weight and bias, adapters cut from larger stacks,
    leading dims, another dtype, rows before the first request."""
    c = case(gpu, 600, 512, 512, 4, 16)
    wide = torch.randn(600, 3 * 512 + 4, device=gpu).to(BF16)
    for off in (0, 512, 5):
        c["x"] = wide[:, off:off + 512]
        check(run(c, [100, 490], [3, 1], gpu, 7), exact(c, [100, 490], [3, 1], first=7))
    c["x"] = c["x"].contiguous()
    want = exact(c, [100, 500], [3, 1])
    w2 = torch.randn(512, 1024, device=gpu).to(BF16)
    w2[:, 256:768] = c["w"]
    check(run(c, [100, 500], [3, 1], gpu, weight=w2[:, 256:768]), want)
    d = dict(c, b=torch.stack([c["b"]] * 3, 1)[:, 1], down=c["down"].transpose(1, 2).contiguous()
             .transpose(1, 2), up=torch.cat([c["up"], c["up"]], 2)[..., :16])
    check(run(d, [100, 500], [3, 1], gpu), want)
    y = run(dict(c, x=c["x"].view(2, 300, 512).float()), [100, 500], [3, 1], gpu)
    assert y.shape == (2, 300, 512) and y.dtype == torch.float32
    check(y.view(600, 512), want)
    assert run(dict(c, x=c["x"][:0]), [], [], gpu).shape == (0, 512)
    check(run(c, [], [], gpu), exact(c, [], []))


def test_lora_linear_without_adapters_is_the_linear(gpu):
    """No adapter: the linear's own bits (rows by the thousand, where both run the same kernel)."""
    from difflet_amd import kernels

    c = case(gpu, 3000, 1024, 2048, 2, 16)
    want = kernels.gemm_call("bf16", c["x"], c["w"], c["b"])
    assert torch.equal(run(c, [1000, 2000], [-1, 7], gpu), want)


def test_lora_linear_keeps_requests_apart(gpu):
    """NaN in one request's rows or one adapter stays with the rows that use it."""
    for rows in (96, 3000):
        c = case(gpu, rows, 512, 512, 3, 16)
        c["down"][2, 3, 5] = float("nan")
        c["up"][1, 17, 2] = float("inf")
        c["x"][5] = float("nan")
        third = rows // 3
        lengths, ids = [third, third, rows - 2 * third], [0, 1, 2]
        y = run(c, lengths, ids, gpu)
        assert bool(y[5].isnan().all()) and bool(y[2 * third:].isnan().all())
        assert not bool(y[third:2 * third, 17].isfinite().any())
        keep = torch.ones_like(y, dtype=torch.bool)
        keep[5], keep[2 * third:], keep[third:2 * third, 17] = False, False, False
        assert bool(y[keep].isfinite().all())


@pytest.mark.parametrize("fmt", ["fp8_rowwise", "mxfp8"])
@pytest.mark.parametrize("rows,k,n,rank", [(1, 1024, 512, 16), (50, 640, 260, 4), (700, 3072, 3072, 64),
                                           (5000, 1024, 3072, 16), (4600, 3072, 4096, 32)])
def test_lora_linear_fp8(gpu, rows, k, n, rank, fmt):
    """An fp8 linear's own result (its kernels' codes and scales, in fp64) and the adapters on the
    unquantized rows."""
    from difflet_amd import kernels
    from difflet_amd.quant.linear import FP8Linear

    c = case(gpu, rows, k, n, 3, rank)
    c["w"][1] = 0  # a channel the linear does not have, which the adapters do
    c["x"][0] = 0
    lin = FP8Linear(k, n, device=gpu, format=fmt)
    lin.load_from_dense_(c["w"], c["b"])
    lin.prepare_kernel_()
    mx = fmt == "mxfp8"
    q, s = kernels.quantize_mxfp8(c["x"], swizzled=True) if mx else kernels.quantize_fp8_rowwise(c["x"])
    wk = lin.weight_kernel.view(torch.float8_e4m3fn)

    def values(codes, scales):
        v = codes.double()
        if mx:
            return (v.view(v.shape[0], -1, 32) * torch.exp2(scales.double() - 127)[..., None]).view(v.shape)
        return v * scales.double()[:, None]

    a, w = values(q, s), values(wk, lin.weight_scale)
    size = a.abs() @ w.abs().t()
    cut = [rows // 2, 0, rows - rows // 2]
    want = exact(c, cut, [1, 0, 2], base=a @ w.t(), extra=size * k * 2.0 ** -24)
    check(run(c, cut, [1, 0, 2], gpu, weight=lin.weight_kernel, weight_scale=lin.weight_scale), want)
    got = kernels.lora_linear("mx" if mx else "fp8", c["x"], wk, c["b"], c["down"], c["up"],
                              c["scale"], starts(cut, gpu),
                              torch.tensor([1, 0, 2], dtype=torch.int32, device=gpu),
                              w_scale=lin.weight_scale, prepared=(q, s))
    check(got, want)


@pytest.mark.parametrize("rows", [12, 700, 4600])
def test_lora_linear_graph_follows_new_requests(gpu, rows):
    c = case(gpu, rows, 1024, 2048, 4, 16)
    st, ids = starts([1, rows - 1], gpu), torch.tensor([0, 1], dtype=torch.int32, device=gpu)
    from difflet_amd.backends.rocm.ops_impl.linear import lora_linear

    def step():
        return lora_linear(c["x"], c["w"], c["b"], c["down"], c["up"], c["scale"], st, ids)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i, (n, a) in enumerate(((1, [0, 1]), (rows // 2, [3, 2]), (rows, [1, -1]), (0, [2, 3]))):
        st.copy_(starts([n, rows - n], gpu))
        ids.copy_(torch.tensor(a, dtype=torch.int32))
        c["x"].copy_(case(gpu, rows, 1024, 2048, 4, 16, seed=9 + i)["x"])
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        check(out, exact(c, [n, rows - n], a))


def test_lora_linear_row_numbers_out_of_order_stay_inside(gpu):
    c = case(gpu, 400, 256, 512, 2, 8)
    from difflet_amd.backends.rocm.ops_impl.linear import lora_linear

    st = torch.tensor([0, 100, -5, 2**31 - 1], dtype=torch.int32, device=gpu)
    ids = torch.tensor([0, 99, -2**31], dtype=torch.int32, device=gpu)
    y = lora_linear(c["x"], c["w"], c["b"], c["down"], c["up"], c["scale"], st, ids)
    assert y.shape == (400, 512)  # no result is promised for them


def test_lora_linear_compiles(gpu):
    c = case(gpu, 70, 256, 512, 2, 8)
    st, ids = starts([30, 40], gpu), torch.tensor([1, 0], dtype=torch.int32, device=gpu)
    from difflet_amd.backends.rocm.ops_impl.linear import lora_linear

    f = lambda x: lora_linear(x * 2, c["w"], c["b"], c["down"], c["up"], c["scale"], st, ids) + 1  # noqa: E731
    assert torch.equal(torch.compile(f, fullgraph=True, backend="aot_eager")(c["x"]), f(c["x"]))


@pytest.mark.parametrize("count", [62, 63, 64, 65])
@pytest.mark.parametrize("length,n", [(5, 512), (41, 512), (300, 1024)])
def test_lora_linear_around_a_wavefront_of_requests(gpu, count, length, n):
    """Tiles of one request, of several and of more requests than a wavefront has lanes."""
    rows = count * length + 3
    c = case(gpu, rows, 256, n, 7, 24)
    ids = [(5 * i) % 8 - 1 for i in range(count)]
    check(run(c, [length] * count, ids, gpu, 2), exact(c, [length] * count, ids, first=2))


@pytest.mark.parametrize("rank", [3, 8, 24, 72, 200])
@pytest.mark.parametrize("k,n", [(512, 1024), (1024, 4096)])
def test_lora_linear_tiles_that_end_with_a_request(gpu, k, n, rank):
    """Requests that fill whole tiles, empty ones on their borders, tiles of no request before, between
    and behind, in launches of few and of many tiles."""
    lengths, ids = [256, 0, 0, 256, 512, 0, 2048, 256], [2, 0, 1, 1, -1, 2, 0, 5]
    for first in (0, 512, 300):
        c = case(gpu, first + sum(lengths) + 600, k, n, 3, rank, seed=first)
        check(run(c, lengths, ids, gpu, first), exact(c, lengths, ids, first=first))


def test_lora_linear_of_one_request_keeps_the_formula(gpu):
    """Rows that all have an adapter with an infinity: it stays in its column; no gradient is made up."""
    for rows in (40, 3000):
        c = case(gpu, rows, 512, 512, 2, 16)
        c["up"][1, 17, 2] = float("inf")
        y = run(c, [rows], [1], gpu)
        assert not bool(y[:, 17].isfinite().any())
        y[:, 17] = 0
        assert bool(y.isfinite().all())
    x = c["x"].clone().requires_grad_()
    with pytest.raises(RuntimeError):
        run(dict(c, x=x), [rows], [1], gpu).sum().backward()
