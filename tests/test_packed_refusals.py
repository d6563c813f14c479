"""What the operators over packed requests refuse, before any device work (no GPU needed)."""

import ctypes

import pytest
import torch

BF16 = torch.bfloat16


def test_rms_norm_quantized_refusals():
    from difflet_amd.backends.rocm.ops_impl.norm import rms_norm_quantized as f

    x = torch.zeros(2, 256, dtype=BF16)
    with pytest.raises(ValueError, match="format"):
        f(x, None, 1e-6, format="fp4")
    with pytest.raises(ValueError, match="device"):
        f(x, None, 1e-6)
    m = torch.zeros(2, 256, dtype=BF16, device="meta")
    with pytest.raises(ValueError, match="device"):
        f(m, None, 1e-6)


def _rms(lib, **kw):
    a = dict(x=16, ldx=256, residual=None, ldr=0, hidden=None, ldh=0, codes=16, ldq=256, scales=16,
             lds=8, dtype=1, rows=1, dim=256, weight=None, wdt=0, eps=1e-6, mx=0)
    a.update(kw)
    return lib.difflet_rocm_rms_norm_quant(*a.values(), None)


def test_rms_norm_quant_entry_point_refusals():
    from difflet_amd import _lib

    lib = _lib.load()
    assert _rms(lib, rows=0) == _lib.OK
    for bad in (dict(dim=12), dict(dim=0), dict(dim=136, mx=1), dict(rows=-1), dict(dtype=3),
                dict(x=None), dict(codes=None), dict(scales=None), dict(hidden=16),
                dict(ldx=255), dict(ldq=248), dict(x=8), dict(codes=12), dict(weight=16, wdt=5),
                dict(mx=1, lds=7), dict(residual=16, ldr=4), dict(residual=16, hidden=16, ldh=128)):
        assert _rms(lib, **bad) == _lib.EINVAL, bad
    assert _rms(lib, dim=16392, ldx=16392, ldq=16392) == _lib.EUNSUPPORTED


def test_rope_axes_refusals():
    from difflet_amd import kernels
    from difflet_amd.backends.rocm.ops_impl.embeddings import apply_rotary_axes as f

    q, pos = torch.zeros(4, 2, 64), torch.zeros(4, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="layout"):
        f(q, None, pos, (64,), layout="pairs")
    with pytest.raises(ValueError, match="device"):
        f(q, None, pos, (64,))
    with pytest.raises(ValueError, match="device"):
        kernels.rope_axes(q[None], None, pos[None], (64,))


def _rope(lib, **kw):
    st = (ctypes.c_int64 * 3)(128, 128, 64)
    a = dict(q=16, qo=16, qs=st, qos=st, qh=2, k=None, ko=None, ks=None, kos=None, kh=0, dtype=1,
             batch=1, seq=1, dim=64, pos=16, pdt=5, pbs=0, axes=1, pairs=32,
             turns=(ctypes.c_double * 128)(), axis=(ctypes.c_uint8 * 128)(), halves=0)
    a.update(kw)
    return lib.difflet_rocm_rope_axes(*a.values(), None)


def test_rope_axes_entry_point_refusals():
    from difflet_amd import _lib

    lib = _lib.load()
    assert _rope(lib, seq=0) == _lib.OK
    assert _rope(lib, qh=0) == _lib.OK
    ones = (ctypes.c_uint8 * 128)(*[1] * 128)
    for bad in (dict(dim=0), dict(axes=0), dict(axes=9), dict(pairs=0), dict(pairs=33),
                dict(pairs=129, dim=512), dict(turns=None), dict(axis=None), dict(axis=ones),
                dict(dtype=3), dict(pdt=1), dict(q=None), dict(qo=None), dict(qs=None),
                dict(kh=1), dict(pos=None), dict(batch=-1)):
        assert _rope(lib, **bad) == _lib.EINVAL, bad


def test_packed_cross_attention_refusals():
    from difflet_amd import kernels
    from difflet_amd.backends.rocm.ops_impl.attention import packed_cross_attention as f

    q, s = torch.zeros(4, 2, 64, dtype=BF16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="device"):
        f(q, q, q, s, s)
    with pytest.raises(ValueError, match="device"):
        kernels.packed_attention(q, q, q, s, s, scale=1.0)


def _attn(lib, **kw):
    st = (ctypes.c_int64 * 2)(128, 64)
    a = dict(q=16, k=16, v=16, o=16, dtype=1, rq=1, rk=1, hk=2, g=1, d=64, qs=st, ks=st, vs=st,
             os=st, qst=16, kst=16, n=1, scale=1.0, zero=1, ws=None, wb=0)
    a.update(kw)
    return lib.difflet_rocm_packed_attention(*a.values(), None)


def test_packed_attention_entry_point_refusals():
    from difflet_amd import _lib

    lib = _lib.load()
    assert _attn(lib, rq=0) == _lib.OK
    odd, far = (ctypes.c_int64 * 2)(124, 64), (ctypes.c_int64 * 2)(1 << 24, 64)
    back = (ctypes.c_int64 * 2)(-128, 64)
    for bad in (dict(hk=0), dict(g=0), dict(rq=-1), dict(n=-1), dict(q=None), dict(k=None),
                dict(o=None), dict(qst=None), dict(kst=None), dict(qs=None), dict(qs=odd),
                dict(ks=odd), dict(q=8), dict(v=24), dict(o=4), dict(scale=float("inf")),
                dict(scale=float("nan"))):
        assert _attn(lib, **bad) == _lib.EINVAL, bad
    for bad in (dict(dtype=0), dict(d=32), dict(ks=far), dict(vs=back), dict(rq=1 << 31),
                dict(hk=65537)):
        assert _attn(lib, **bad) == _lib.EUNSUPPORTED, bad
    size = lib.difflet_rocm_packed_attention_workspace_bytes
    assert size(16, 32000, 16, 4, 7, 128) > 0  # single tokens: keys in pieces
    assert size(40000, 738, 2, 40, 1, 128) == 0 and size(0, 1, 1, 1, 1, 64) == 0


def test_lora_linear_refusals():
    from difflet_amd import kernels
    from difflet_amd.backends.rocm.ops_impl.linear import lora_linear as f

    x, w = torch.zeros(4, 64, dtype=BF16), torch.zeros(8, 64, dtype=BF16)
    down, up = torch.zeros(1, 4, 64, dtype=BF16), torch.zeros(1, 8, 4, dtype=BF16)
    one, s = torch.ones(1), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="device"):
        f(x, w, None, down, up, one, s, s[:1])
    with pytest.raises(ValueError, match="device"):
        kernels.lora_linear("bf16", x, w, None, down, up, one, s, s[:1])


def _lora(lib, **kw):
    a = dict(kind=0, a=16, lda=64, a_scale=None, w=16, ldw=64, w_scale=None, bias=None, c=16, ldc=8,
             m=1, n=8, k=64, x=16, ldx=64, x_cols=64, down=16, up=16, up_rows=8, scale=16, adapters=1,
             rank=4, starts=16, ids=16, requests=1, ws=256, wb=1 << 20)
    a.update(kw)
    return lib.difflet_rocm_lora_linear(*a.values(), None)


def test_lora_entry_point_refusals():
    from difflet_amd import _lib

    lib = _lib.load()
    assert _lora(lib, m=0) == _lib.OK
    for bad in (dict(kind=3), dict(m=-1), dict(n=0), dict(rank=0), dict(x_cols=72), dict(x_cols=60),
                dict(x_cols=0), dict(up_rows=9), dict(up_rows=0), dict(x=None), dict(starts=None),
                dict(ids=None), dict(down=None), dict(up=None), dict(scale=None), dict(ldx=56),
                dict(x=8), dict(down=8), dict(ws=None), dict(wb=16), dict(ws=128),
                dict(adapters=-1), dict(requests=-1)):
        assert _lora(lib, **bad) == _lib.EINVAL, bad
    assert _lora(lib, rank=1025) == _lib.EUNSUPPORTED
    assert lib.difflet_rocm_lora_workspace_bytes(0, 0, 8, 64, 4, 1) == 0
    assert lib.difflet_rocm_lora_workspace_bytes(5, 1, 8, 64, 4, 1) == 0
