"""What the E4M3 operators refuse, on the host and before anything is launched."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from plaquant_b200 import _lib, build
    build.build_library()
    build.build_torch_front_end()
    return _lib.lib()


@pytest.fixture(scope="module")
def p16():
    buf = (ctypes.c_uint8 * 8192)()
    p16._keep = buf
    return (ctypes.addressof(buf) + 15) & ~15


SHAPE, NULL, ALIGN, LIMIT = -2, -1, -3, -7


def test_quantisers(lib, p16):
    pack = lambda **k: lib.plq_fp8_pack(*{**dict(x=p16, ldx=256, res=None, ldr=0, h=None, gamma=None, eps=1e-6, rows=2, k=256, codes=p16, scales=p16, stream=None), **k}.values())  # noqa: E731
    assert pack(k=250) == SHAPE and pack(k=0) == SHAPE and pack(rows=-1) == SHAPE
    assert pack(ldx=128) == SHAPE and pack(ldx=260) == SHAPE
    assert pack(k=32784, ldx=32784) == LIMIT and pack(rows=1 << 31) == LIMIT
    assert pack(res=p16, ldr=256, h=p16) == NULL                  # a residual without a norm
    assert pack(res=p16, ldr=256, gamma=p16) == NULL and pack(res=p16, ldr=8, h=p16, gamma=p16) == SHAPE
    assert pack(x=None) == NULL and pack(codes=None) == NULL and pack(scales=None) == NULL
    assert pack(x=p16 + 2) == ALIGN and pack(codes=p16 + 8) == ALIGN and pack(scales=p16 + 2) == ALIGN and pack(gamma=p16 + 2) == ALIGN
    assert pack(rows=0, x=None) == 0
    assert lib.plq_fp8_pack_weight(p16, 4, 24, p16, p16, None) == SHAPE
    assert lib.plq_fp8_pack_weight(p16, 128 * 65536, 16, p16, p16, None) == LIMIT
    assert lib.plq_fp8_pack_weight(None, 4, 32, p16, p16, None) == NULL
    assert lib.plq_fp8_unpack(p16, p16, 4, 32, 64, p16, None) == SHAPE
    assert lib.plq_fp8_unpack(p16, p16, 4, 32, 1, None, None) == NULL


def test_product(lib, p16):
    gemm = lambda **k: lib.plq_fp8_gemm(*{**dict(a=p16, sa=p16, w=p16, sw=p16, m=4, n=8, k=32, y=p16, ldy=8, f32=0, status=p16, flags=0, stream=None), **k}.values())  # noqa: E731
    assert gemm(m=0) == SHAPE and gemm(n=0) == SHAPE and gemm(k=24) == SHAPE and gemm(k=0) == SHAPE and gemm(ldy=7) == SHAPE
    assert gemm(flags=9 << 4) == SHAPE and gemm(flags=-16) == SHAPE
    assert gemm(m=(1 << 30) + 1) == LIMIT and gemm(n=(1 << 30) + 1, ldy=1 << 31) == LIMIT and gemm(k=1 << 25) == LIMIT
    for name in ("a", "sa", "w", "sw", "y", "status"):
        assert gemm(**{name: None}) == NULL
    assert gemm(a=p16 + 8) == ALIGN and gemm(w=p16 + 1) == ALIGN and gemm(sa=p16 + 2) == ALIGN and gemm(y=p16 + 1) == ALIGN and gemm(y=p16 + 2, f32=1) == ALIGN


def test_cache(lib, p16):
    append = lambda **k: lib.plq_rope_kv_append_fp8(*{**dict(qkv=p16, ld=512, cos=p16, sin=p16, cs=0, b=1, t=2, heads=2, kv_heads=1, q=p16, kc=p16, ks=p16, vc=p16,  # noqa: E731
                                                             vs=p16, t_max=64, dev=None, each=0, pos=0, status=p16, stream=None), **k}.values())
    assert append(heads=0) == SHAPE and append(kv_heads=0) == SHAPE and append(ld=384) == SHAPE and append(ld=516) == SHAPE and append(t_max=0) == SHAPE
    assert append(pos=63) == SHAPE and append(t=65) == SHAPE and append(cs=-4) == SHAPE and append(cs=130) == SHAPE
    assert append(heads=4095, ld=1 << 20) == LIMIT and append(t_max=1 << 31) == LIMIT
    assert append(t=0, qkv=None) == 0 and append(b=0) == 0
    for name in ("qkv", "cos", "sin", "q", "kc", "ks", "vc", "vs"):
        assert append(**{name: None}) == NULL
    assert append(kc=p16 + 4) == ALIGN and append(ks=p16 + 2) == ALIGN and append(dev=p16 + 4) == ALIGN
    attend = lambda **k: lib.plq_fp8_attention(*{**dict(q=p16, kc=p16, ks=p16, vc=p16, vs=p16, b=1, t=1, heads=4, kv_heads=2, t_max=64, dev=None, each=0, pos=5, ctx=6,  # noqa: E731
                                                        scale=1.0, out=p16, ws=None, ws_bytes=0, status=p16, stream=None), **k}.values())
    assert attend(heads=3) == SHAPE and attend(kv_heads=0) == SHAPE and attend(pos=64) == SHAPE and attend(ctx=5) == SHAPE and attend(ctx=65) == SHAPE
    assert attend(b=65536) == LIMIT and attend(t_max=1 << 31, ctx=64) == LIMIT and attend(heads=4098) == LIMIT
    assert attend(b=0) == 0 and attend(t=0) == 0
    for name in ("q", "kc", "ks", "vc", "vs", "out"):
        assert attend(**{name: None}) == NULL
    assert attend(q=p16 + 2) == ALIGN and attend(out=p16 + 8) == ALIGN
    assert lib.plq_fp8_attention_workspace_bytes(0, 1, 4, 2, 64) == 0 and lib.plq_fp8_attention_workspace_bytes(1, 1, 3, 2, 64) == 0


def test_python_checks_need_no_gpu(lib):
    from plaquant_b200 import kv_cache, ops
    from plaquant_b200.quantize import Fp8Linear
    bf = torch.bfloat16
    x, g = torch.zeros(2, 32, dtype=bf), torch.ones(32, dtype=bf)
    u8, f32 = torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 1)
    a, w = ops.Fp8Matrix(u8, f32, 1), ops.Fp8Matrix(u8, f32[:1], 128)
    cache = kv_cache.Fp8Cache.empty(1, 64, 2, "cpu")
    calls = [lambda: ops.fp8_pack(x), lambda: ops.add_rmsnorm_fp8_pack(x, x, g, 1e-6), lambda: ops.fp8_pack_weight(x), lambda: ops.fp8_unpack(a),
             lambda: ops.fp8_gemm(a, w), lambda: Fp8Linear(u8, f32[:1])(x),
             lambda: ops.rope_kv_append_fp8(torch.zeros(1, 1, 8 * 128, dtype=bf), torch.zeros(128), torch.zeros(128), 4, 2, cache, 0),
             lambda: ops.fp8_cache_attention(torch.zeros(1, 1, 4, 128, dtype=bf), cache, 0)]
    for call in calls:
        with pytest.raises(RuntimeError):                 # no CPU path
            call()
    with pytest.raises(ValueError):
        Fp8Linear(torch.zeros(4, 24, dtype=torch.uint8), torch.zeros(1, 1))
    with pytest.raises(ValueError):
        Fp8Linear(u8, torch.zeros(1, 2))
    with pytest.raises(TypeError):
        ops.add_rmsnorm_fp8_pack(x, x[:1], g, 1e-6)


@pytest.mark.parametrize("change", [dict(k=torch.zeros(1, 64, 2, 64, dtype=torch.uint8)), dict(v=torch.zeros(1, 63, 2, 128, dtype=torch.uint8)),
                                    dict(k=torch.zeros(1, 64, 2, 128)), dict(k_scale=torch.zeros(1, 2, 2)), dict(v_scale=torch.zeros(1, 2, 1, dtype=torch.float64)),
                                    dict(v=torch.zeros(1, 64, 4, 128, dtype=torch.uint8)[:, :, ::2]), dict(v_scale=torch.zeros(1, 1, 2).transpose(1, 2)[:, :, :1].expand(1, 2, 1)[:, ::2].expand(1, 2, 1))])
def test_malformed_caches_are_refused(change):
    from dataclasses import replace
    from plaquant_b200 import kv_cache
    good = kv_cache.Fp8Cache.empty(1, 64, 2, "cpu")
    good.check(1, 2, torch.device("cpu"))
    for bad in ((2, 2), (1, 4)):
        with pytest.raises(TypeError):
            good.check(*bad, torch.device("cpu"))
    with pytest.raises(RuntimeError):
        good.check(1, 2, torch.device("cuda", 0))
    with pytest.raises(TypeError):
        replace(good, **change).check(1, 2, torch.device("cpu"))
