"""RMSNorm with a residual to 8 bits and rotary embedding from positions on several axes, on the
GPU against plain implementations in 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3_STEP = 2.0 ** -4  # half a step of e4m3, relative


def swizzle(k, dev):
    """Position r * 4 + j of a 512-wide tile (or the remainder) is its element j * tile / 4 + r."""
    parts = [torch.arange(t, min(t + 512, k)).view(4, -1).t().reshape(-1) for t in range(0, k, 512)]
    return torch.cat(parts).to(dev)


def check_codes(y, codes, scales, mx):
    """codes and scales against fp64 y [rows, dim]. fp32 errors of y: its sums run over at most 96
    squares a thread and 8 levels between threads, 104 * 2^-24 halved by the root, and a few 2^-24
    more: under 2^-16 in all. A value is then off by half a step of e4m3 (2^-4 of itself, or of
    its smallest normal, 2^-6, of the scale) and those."""
    dev = y.device
    rows, dim = y.shape
    if mx:
        y = y[:, swizzle(dim, dev)].view(rows, -1, 32)
        top = y.abs().amax(-1)
        e = torch.frexp(top)[1].double() - 1
        want = torch.where(top == 0, torch.zeros_like(e), (e + 127 - 7).clamp(0, 255))
        edge = (torch.frexp(top * (1 + 2.0 ** -16))[1] != torch.frexp(top * (1 - 2.0 ** -16))[1])
        assert bool(((scales.double() == want) | edge).all())
        s = torch.exp2(scales.double() - 127)[..., None]
        v = codes.double().view(rows, -1, 32) * s
    else:
        want = y.abs().amax(-1).clamp_min(2.0 ** -112) / 448
        assert bool(((scales.double() - want).abs() <= want * 2.0 ** -16).all())
        s = scales.double()[:, None]
        v = codes.double() * s
    tol = y.abs() * (E4M3_STEP + 2.0 ** -15) + s * 2.0 ** -10 * (1 + 2.0 ** -15)
    bad = (v - y).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float((v - y).abs().max()))


def norm_case(gpu, dtype, rows, dim, seed=0, weight=True):
    g = torch.Generator(device=gpu).manual_seed(seed)
    x = torch.randn(rows, dim, generator=g, device=gpu)
    x[:, ::29] *= 12
    r = torch.randn(rows, dim, generator=g, device=gpu) * 2
    w = (1 + 0.3 * torch.randn(dim, generator=g, device=gpu)).to(dtype) if weight else None
    return x.to(dtype), r.to(dtype), w


def norm_exact(x, r, w, eps):
    h = x.double() + (0 if r is None else r.double())
    y = h / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + eps)
    return h, y if w is None else y * w.double()


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,dim", [(1, 4096), (3, 128), (5, 640), (2, 16384), (1024, 128),
                                      (1025, 4096), (1500, 5120), (1030, 6144), (1100, 896),
                                      (7, 8064)])
def test_rms_norm_quantized_matches_64_bits(gpu, rows, dim, dtype, mx):
    from difflet_amd.backends.rocm.ops_impl.norm import rms_norm_quantized

    x, r, w = norm_case(gpu, dtype, rows, dim, seed=rows + dim)
    fmt = "mxfp8" if mx else "fp8_rowwise"
    codes, scales, hidden = rms_norm_quantized(x, w, 1e-6, residual=r, format=fmt)
    h, y = norm_exact(x, r, w, 1e-6)
    check_codes(y, codes, scales, mx)
    # one fp32 sum, one rounding to the dtype
    assert bool(((hidden.double() - h).abs() <= h.abs() * (torch.finfo(dtype).eps / 2 + 2.0 ** -23)
                 + torch.finfo(dtype).smallest_normal).all())
    codes, scales, same = rms_norm_quantized(x, None, 1e-6, format=fmt)
    assert same is x
    check_codes(norm_exact(x, None, None, 1e-6)[1], codes, scales, mx)


@pytest.mark.parametrize("dim", [8, 24, 136, 1000, 2056, 6152, 12296])
def test_rms_norm_quantized_odd_widths(gpu, dim):
    from difflet_amd.backends.rocm.ops_impl.norm import rms_norm_quantized

    for rows in (3, 1031):
        x, r, w = norm_case(gpu, BF16, rows, dim, seed=dim)
        codes, scales, _ = rms_norm_quantized(x, w.float(), 1e-5, residual=r)
        check_codes(norm_exact(x, r, w, 1e-5)[1], codes, scales, False)


def test_rms_norm_quantized_strides_in_place_and_leading_dims(gpu):
    from difflet_amd import kernels
    from difflet_amd.backends.rocm.ops_impl.norm import rms_norm_quantized

    buf, res, w = norm_case(gpu, BF16, 2 * 9, 3 * 256)
    x, r = buf[:, 256:512], res[:, 5:261]  # rows of a wider buffer; rows off 16 bytes
    codes, scales, hidden = rms_norm_quantized(x.reshape(2, 9, 256), w[:256], 1e-6,
                                               residual=r.reshape(2, 9, 256), format="mxfp8")
    assert codes.shape == (2, 9, 256) and scales.shape == (2, 9, 8) and hidden.shape == (2, 9, 256)
    h, y = norm_exact(x, r, w[:256], 1e-6)
    check_codes(y, codes.reshape(18, 256), scales.reshape(18, 8), True)
    xt = buf[:, :256].t().contiguous().t()  # columns contiguous, rows not
    codes, scales, _ = rms_norm_quantized(xt, w[:256], 1e-6)
    check_codes(norm_exact(xt, None, w[:256], 1e-6)[1], codes, scales, False)
    x2, r2 = x.contiguous(), res[:, 256:512].contiguous()
    want = kernels.rms_norm_quant(x2, w[:256], 1e-6, residual=r2)
    got = kernels.rms_norm_quant(x2, w[:256], 1e-6, residual=r2, hidden=r2)  # over the residual
    assert got[2].data_ptr() == r2.data_ptr()
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("mx", [False, True])
def test_rms_norm_quantized_zero_rows_nan_and_no_rows(gpu, mx):
    from difflet_amd.backends.rocm.ops_impl.norm import rms_norm_quantized

    fmt = "mxfp8" if mx else "fp8_rowwise"
    for rows in (4, 1200):
        x, r, w = norm_case(gpu, BF16, rows, 1024)
        x[0], r[0] = 0, 0
        x[1, 7] = float("nan")
        x[2, 9] = float("inf")
        codes, scales, _ = rms_norm_quantized(x, w, 1e-6, residual=r, format=fmt)
        assert float(codes[0].float().abs().max()) == 0
        assert bool(codes[1].float().isnan().all())
        if mx:
            assert bool((scales[1] == 255).all())
            block = int((swizzle(1024, "cpu") == 9).nonzero()) // 32
            assert int((scales[2] == 255).sum()) == 1 and int(scales[2, block]) == 255
        else:
            assert bool(scales[1:3].isnan().all()) and bool(codes[2].float().isnan().all())
        check_codes(norm_exact(x, r, w, 1e-6)[1][3:], codes[3:], scales[3:], mx)
    codes, scales, hidden = rms_norm_quantized(x[:0], w, 1e-6, residual=r[:0], format=fmt)
    assert codes.shape == (0, 1024) and scales.shape[0] == 0 and hidden.shape == (0, 1024)


# ---------------------------------------------------------------------------------- rotary
def rope_exact(x, positions, axes, theta, halves, shared):
    b, s, h, d = x.shape
    total, ang, done = sum(axes), [], 0
    pos = positions.double().expand(b, s, len(axes)).cpu()
    for a, n in enumerate(axes):
        for j in range(n // 2):
            f = theta ** (-2.0 * (done + j) / total if shared else -2.0 * j / n)
            ang.append(pos[..., a] * f)
        done += n // 2
    ang = torch.stack(ang, -1).to(x.device)[:, :, None]
    c, sn = ang.cos(), ang.sin()
    r = x.double()[..., :total]
    if halves:
        p, q = r[..., : total // 2], r[..., total // 2:]
        y = torch.cat([p * c - q * sn, q * c + p * sn], -1)
        size = torch.cat([p.abs() + q.abs()] * 2, -1)
    else:
        p, q = r[..., 0::2], r[..., 1::2]
        y = torch.stack([p * c - q * sn, q * c + p * sn], -1).flatten(-2)
        size = torch.stack([p.abs() + q.abs()] * 2, -1).flatten(-2)
    rest = x.double()[..., total:]
    return torch.cat([y, rest], -1), torch.cat([size, 0 * rest], -1)


def check_rope(got, x, positions, axes, theta, halves, shared):
    """Angles: a fraction of a turn rounded to fp32 (half a turn at most, 2^-25 of it, pi 2^-24 in
    radians) and sine and cosine of two units in the last place: under 2^-21 of |a| + |b|, and one
    rounding to the dtype."""
    y, size = rope_exact(x, positions, axes, theta, halves, shared)
    tol = size * 2.0 ** -21 + y.abs() * torch.finfo(x.dtype).eps / 2 + 1e-7 * (x.dtype == F16)
    assert got.dtype == x.dtype and got.shape == x.shape
    bad = (got.double() - y).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float((got.double() - y).abs().max()))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("axes,dim,shared", [((16, 56, 56), 128, False), ((44, 42, 42), 128, False),
                                             ((32, 48, 48), 128, True), ((64,), 64, False),
                                             ((20, 12), 80, False), ((32, 32), 96, True),
                                             ((6, 4, 2), 14, False), ((2,) * 8, 17, True)])
def test_rope_axes_matches_64_bits(gpu, axes, dim, shared, halves, dtype):
    from difflet_amd.backends.rocm.ops_impl.embeddings import apply_rotary_axes

    g = torch.Generator(device=gpu).manual_seed(dim)
    for b, s, h, hk, far in ((1, 1, 3, 1, 1 << 21), (2, 77, 6, 2, 1000), (1, 2300, 2, 2, 64)):
        q = torch.randn(b, s, h, dim, generator=g, device=gpu).to(dtype)
        k = torch.randn(b, s, hk, dim, generator=g, device=gpu).to(dtype)
        pos = torch.randint(-far, far, (b, s, len(axes)), generator=g, device=gpu)
        qo, ko = apply_rotary_axes(q, k, pos, axes, layout="halves" if halves else "interleaved",
                                   shared_frequencies=shared)
        for got, x in ((qo, q), (ko, k)):
            check_rope(got, x, pos, axes, 1e4, halves, shared)


@pytest.mark.parametrize("halves", [False, True])
def test_rope_axes_strides_positions_and_in_place(gpu, halves):
    from difflet_amd import kernels
    from difflet_amd.backends.rocm.ops_impl.embeddings import apply_rotary_axes

    axes, layout = (16, 24, 24), "halves" if halves else "interleaved"
    g = torch.Generator(device=gpu).manual_seed(1)
    buf = torch.randn(2, 50, 9 * 64 + 3, generator=g, device=gpu).to(BF16)
    pos = torch.randint(0, 5000, (1, 50, 3), generator=g, device=gpu)
    for off in (0, 3):  # heads on 16 bytes or not, in a fused projection's rows of an odd width
        q = buf[..., off:off + 5 * 64].unflatten(-1, (5, 64))
        k = buf[..., off + 5 * 64:off + 7 * 64].unflatten(-1, (2, 64))
        for p in (pos, pos.to(torch.int32), pos.float(), pos.expand(2, 50, 3)):
            qo, ko = apply_rotary_axes(q, k, p, axes, theta=500.0, layout=layout)
            check_rope(qo, q, p, axes, 500.0, halves, False)
            check_rope(ko, k, p, axes, 500.0, halves, False)
    x = torch.randn(2, 5, 50, 64, generator=g, device=gpu).to(F16).transpose(1, 2)  # [B, H, S, D]
    qo, none = apply_rotary_axes(x, None, pos, axes, layout=layout)
    assert none is None
    check_rope(qo, x, pos, axes, 1e4, halves, False)
    qo, ko = apply_rotary_axes(x[0], x[1], pos[0], axes, layout=layout)  # no batch
    check_rope(qo[None], x[:1], pos, axes, 1e4, halves, False)
    check_rope(ko[None], x[1:], pos, axes, 1e4, halves, False)
    want = apply_rotary_axes(q, k, pos, axes, layout=layout)
    before = buf.clone()
    kernels.rope_axes(q, k, pos, axes, halves=halves, q_out=q, k_out=k)  # over the projection
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    buf[..., 3:3 + 7 * 64] = before[..., 3:3 + 7 * 64]
    assert torch.equal(buf, before)  # nothing else was written


def test_rope_axes_far_positions_and_empty(gpu):
    from difflet_amd.backends.rocm.ops_impl.embeddings import apply_rotary_axes

    q = torch.randn(1, 6, 2, 64, device=gpu)
    pos = torch.tensor([0, 1, 2**31 - 1, 2**40 + 1, -2**45, 2**24 + 1], device=gpu).view(1, 6, 1)
    got, _ = apply_rotary_axes(q[:, :3], None, pos[:, :3], (64,))
    check_rope(got, q[:, :3], pos[:, :3], (64,), 1e4, False, False)
    got, _ = apply_rotary_axes(q, None, pos, (64,))
    n = got.double().square().sum(-1) / q.double().square().sum(-1)
    assert float((n - 1).abs().max()) < 2.0 ** -20  # still a rotation
    empty, _ = apply_rotary_axes(q[:, :0], None, pos[:, :0], (64,))
    assert empty.shape == (1, 0, 2, 64)


def test_packed_rows_operators_replay_in_a_graph(gpu):
    """Captured together and replayed with new inputs between eager work, on a stream of its own."""
    from difflet_amd.backends.rocm.ops_impl.embeddings import apply_rotary_axes
    from difflet_amd.backends.rocm.ops_impl.norm import rms_norm_quantized

    x, r, w = norm_case(gpu, BF16, 700, 1024)
    pos = torch.zeros(1, 700, 2, dtype=torch.int32, device=gpu)

    def step():
        codes, scales, h = rms_norm_quantized(x, w, 1e-6, residual=r)
        q, _ = apply_rotary_axes(h.view(1, 700, 8, 128), None, pos, (64, 64))
        return codes, scales, h, q

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.copy_(norm_case(gpu, BF16, 700, 1024, seed=10 + i)[0])
        pos.copy_(torch.randint(0, 9999, pos.shape, device=gpu))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_packed_rows_operators_make_up_no_gradient(gpu):
    from difflet_amd.backends.rocm.ops_impl.embeddings import apply_rotary_axes
    from difflet_amd.backends.rocm.ops_impl.norm import rms_norm_quantized

    x, r, w = norm_case(gpu, BF16, 9, 256)
    x.requires_grad_()
    with pytest.raises(RuntimeError):
        rms_norm_quantized(x, w, 1e-6, residual=r)[2].float().sum().backward()
    pos = torch.zeros(9, 1, dtype=torch.int32, device=gpu)
    with pytest.raises(RuntimeError):
        apply_rotary_axes(x.view(9, 2, 128), None, pos, (64,))[0].float().sum().backward()
