"""E4M3 quantisers (a scale per 128 columns of a row, or per 128 x 128 weights) and their product, against float64."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 1e-6


@pytest.fixture(scope="module")
def plq():
    import plaquant_b200
    return plaquant_b200


def _rand(shape, seed, gain=1.0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * gain
    if shape[-1] > 50:
        x[..., torch.randperm(shape[-1], generator=g)[: shape[-1] // 50]] *= 20.0
    return x.to(dtype).cuda()


def _pad_blocks(y):
    k = y.shape[-1]
    n = -(-k // 128)
    return torch.nn.functional.pad(y, (0, n * 128 - k)).unflatten(-1, (n, 128))


def _codes_of(y):
    """Codes and scales of float32 rows by the definition, in the kernel's operations: equal to the last bit.  (Divisions by
    a tensor: PyTorch turns a division by a Python number into a product with its rounded reciprocal.)"""
    b = _pad_blocks(y)
    a = b.abs().amax(-1).clamp_min(2.0 ** -100)
    codes = (b * (torch.full_like(a, 448.0) / a)[..., None]).to(torch.float8_e4m3fn)
    return codes.flatten(-2).view(torch.uint8)[..., : y.shape[-1]], a / torch.full_like(a, 448.0)


def _values(codes, scales):
    k = codes.shape[-1]
    v = _pad_blocks(codes.contiguous().view(torch.float8_e4m3fn).double()) * scales.double()[..., None]
    return v.flatten(-2)[..., :k]


def _check_quantised(p, y):
    """`y` float64: every value within half a step of its code (relative 2^-4, or 2^-10 of the scale near zero; 2^-10 of that
    for float32 arithmetic in front of the rounding), every scale within a few float32 roundings."""
    top = _pad_blocks(y).abs().amax(-1).clamp_min(2.0 ** -100)
    assert torch.all((p.scales.double() * 448.0 / top - 1).abs() <= 2.0 ** -20)
    step = torch.maximum(y.abs() * 2.0 ** -4, (p.scales.double() * 2.0 ** -10).repeat_interleave(128, -1)[..., : y.shape[-1]])
    assert torch.all((_values(p.codes, p.scales) - y).abs() <= step * (1 + 2.0 ** -10))


@pytest.mark.parametrize("rows,k", [(1, 16), (3, 128), (1, 144), (7, 1040), (5, 4096), (2, 4112), (33, 8192), (3, 12288), (2, 28672), (2, 32768)])
def test_rows_without_a_norm_bit_exact(plq, rows, k):
    x = _rand((rows, k), 1)
    p = plq.ops.fp8_pack(x)
    codes, scales = _codes_of(x.float())
    assert torch.equal(p.codes, codes) and torch.equal(p.scales, scales)
    assert torch.equal(plq.ops.fp8_unpack(p), (_pad_blocks(p.codes.view(torch.float8_e4m3fn).float()) * p.scales[..., None]).flatten(-2)[:, :k].to(torch.bfloat16))


@pytest.mark.parametrize("rows,k", [(1, 16), (1, 4096), (333, 4112), (3, 144), (64, 8192), (2, 16400), (3, 32768)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_and_residual(plq, rows, k, residual):
    x, r, gamma = _rand((rows, k), 2), _rand((rows, k), 3), _rand((k,), 4)
    if residual:
        h, p = plq.ops.add_rmsnorm_fp8_pack(x, r, gamma, EPS)
        assert torch.equal(h, r + x)
    else:
        h, p = x, plq.ops.fp8_pack(x, gamma=gamma, eps=EPS)
    f = h.double()
    _check_quantised(p, gamma.double() * f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS))


@pytest.mark.parametrize("n,k", [(1, 16), (128, 128), (129, 144), (300, 1040), (4096, 512)])
def test_weights_bit_exact(plq, n, k):
    w = _rand((n, k), 5, 0.02)
    p = plq.ops.fp8_pack_weight(w)
    nb, kb = -(-n // 128), -(-k // 128)
    b = torch.nn.functional.pad(w.float(), (0, kb * 128 - k, 0, nb * 128 - n)).view(nb, 128, kb, 128)
    a = b.abs().amax((1, 3)).clamp_min(2.0 ** -100)
    codes = (b * (torch.full_like(a, 448.0) / a)[:, None, :, None]).view(nb * 128, kb * 128)[:n, :k].to(torch.float8_e4m3fn)
    assert torch.equal(p.codes, codes.view(torch.uint8)) and torch.equal(p.scales, a / torch.full_like(a, 448.0))
    full = p.scales.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    assert torch.equal(plq.ops.fp8_unpack(p), (p.codes.view(torch.float8_e4m3fn).float() * full).to(torch.bfloat16))


def test_rows_of_views_and_slices(plq):
    """Rows further apart than they are long, transposed and misaligned ones, a leading shape, no rows."""
    x = _rand((6, 3, 512), 6)
    want = _codes_of(x.float().reshape(18, 512))
    for view in (x, x.transpose(0, 1).contiguous().transpose(0, 1)):
        p = plq.ops.fp8_pack(view)
        assert torch.equal(p.codes, want[0]) and torch.equal(p.scales, want[1])
    for view in (x[:, 1], x[:, -1:], x[..., 8:264], x[..., 1:257], x[:, 0].t().contiguous().t()):
        flat = view.reshape(-1, view.shape[-1])
        p = plq.ops.fp8_pack(view)
        codes, scales = _codes_of(flat.float())
        assert torch.equal(p.codes, codes) and torch.equal(p.scales, scales)
    p = plq.ops.fp8_pack(x[:0])
    assert p.rows == 0 and tuple(p.scales.shape) == (0, 4)
    gamma = _rand((512,), 7)
    h, p = plq.ops.add_rmsnorm_fp8_pack(x[:, -1:], x[:, :1], gamma, EPS)
    h2, p2 = plq.ops.add_rmsnorm_fp8_pack(x[:, -1:].contiguous(), x[:, :1].contiguous(), gamma, EPS)
    assert h.shape == (6, 1, 512) and torch.equal(h, h2) and torch.equal(p.codes, p2.codes) and torch.equal(p.scales, p2.scales)


def test_zero_tiny_and_not_finite_blocks(plq):
    x = torch.zeros(4, 384, dtype=torch.bfloat16, device="cuda")
    x[0, 5], x[1, 130], x[2, 1], x[3, 383] = float("nan"), float("inf"), 1e-38, -3e38
    p = plq.ops.fp8_pack(x)
    v = plq.ops.fp8_unpack(p)
    nan = torch.zeros(4, 3, dtype=torch.bool, device="cuda")
    nan[0, 0] = nan[1, 1] = True
    assert torch.equal(p.scales.isnan(), nan) and torch.equal(v.isnan(), nan.repeat_interleave(128, 1))
    assert torch.all(p.codes[nan.repeat_interleave(128, 1)] == 0)
    assert torch.all(v[~nan.repeat_interleave(128, 1) & (x.abs() < 1)] == 0)          # 1e-38 is below a step of the smallest scale
    assert abs(float(v[3, 383]) / -3e38 - 1) <= 2.0 ** -7
    # a row that is not finite is NaN in all of its blocks behind a norm
    p = plq.ops.fp8_pack(x, gamma=torch.ones(384, dtype=torch.bfloat16, device="cuda"))
    assert torch.equal(p.scales.isnan().all(1), torch.tensor([True, False, False, False], device="cuda"))


def _operands(m, n, k, seed):
    import plaquant_b200 as plq
    return plq.ops.fp8_pack(_rand((m, k), seed)), plq.ops.fp8_pack_weight(_rand((n, k), seed + 1, 0.02))


def _check_product(y, a, w):
    """Each K block's 128 products are added by the tensor core, the blocks by float32 multiply-adds: at most one unit of 2^-23
    of the sum of magnitudes per addition (2^-23, not 2^-24: the tensor core may cut where float32 rounds); scales 2^-23."""
    n, k = w.rows, w.k
    av = _values(a.codes, a.scales)
    wv = w.codes.view(torch.float8_e4m3fn).double() * w.scales.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    want = av @ wv.t()
    bound = (av.abs() @ wv.abs().t()) * ((min(k, 128) + -(-k // 128) + 3) * 2.0 ** -23)
    if y.dtype == torch.bfloat16:
        bound = bound + (want.abs() + bound) * 2.0 ** -8
    err = (y.double() - want).abs()
    assert torch.all(err <= bound + 1e-37), float((err - bound).max())


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("n,k", [(1, 16), (128, 128), (200, 400), (1000, 2064), (4097, 512)])
def test_product_of_a_few_rows(plq, m, n, k):
    a, w = _operands(m, n, k, 10 * m + n)
    for dtype in (torch.bfloat16, torch.float32):
        _check_product(plq.ops.fp8_gemm(a, w, out_dtype=dtype), a, w)
        _check_product(plq.ops.fp8_gemm(a, w, out_dtype=dtype, variant="rows"), a, w)
    plq.check_device_status()


@pytest.mark.parametrize("variant", ["128x128", "pair256x256", "pair256x128"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (65, 100, 128), (128, 128, 400), (129, 257, 1040), (300, 1001, 2064), (513, 768, 1024), (256, 5000, 272),
                                   (20, 300, 4112), (130, 1500, 8192)])
def test_product_of_many_rows(plq, variant, m, n, k):
    a, w = _operands(m, n, k, m + n)
    for dtype in (torch.bfloat16, torch.float32):
        _check_product(plq.ops.fp8_gemm(a, w, out_dtype=dtype, variant=variant), a, w)
    plq.check_device_status()


@pytest.mark.parametrize("m,n,k", [(77, 6144, 4096), (16, 8192, 8192), (1, 20000, 4096), (2000, 4096, 1024), (4096, 2048, 512)])
def test_product_of_ordinary_sizes(plq, m, n, k):
    a, w = _operands(m, n, k, m)
    y = plq.ops.fp8_gemm(a, w)
    _check_product(y, a, w)
    assert torch.equal(y, plq.ops.fp8_gemm(a, w, static_weights=True))        # the same sums in the same order
    plq.check_device_status()


def test_product_into_a_buffer(plq):
    """Only the rows and columns of the result are written, at any row stride and alignment."""
    for m, n, k in ((5, 37, 256), (130, 100, 256), (70, 129, 128)):
        a, w = _operands(m, n, k, 3)
        want = plq.ops.fp8_gemm(a, w)
        for stride, shift in ((n, 0), (n + 3, 1), (n + 16 - n % 16, 0), (2 * n, 8)):
            store = torch.full((m * stride + shift + 8,), 7.0, dtype=torch.bfloat16, device="cuda")
            out = store[shift: shift + m * stride].view(m, stride)[:, :n]
            assert plq.ops.fp8_gemm(a, w, out=out) is out
            assert torch.equal(out, want)
            store[shift: shift + m * stride].view(m, stride)[:, :n] = 7.0
            assert torch.all(store == 7.0)
    a, w = _operands(3, 16, 128, 4)
    empty = plq.ops.Fp8Matrix(a.codes[:0], a.scales[:0], 1)
    assert tuple(plq.ops.fp8_gemm(empty, w).shape) == (0, 16)


@pytest.mark.parametrize("variant", ["128x128", "pair256x256", "pair256x128"])
@pytest.mark.parametrize("m,n", [(129, 258), (200, 301), (33, 70), (257, 15), (64, 500)])
def test_many_rows_at_any_edge_and_alignment(plq, variant, m, n):
    """Rows that allow stores of 32, 16, four and two bytes, both types, edges inside a group of 16 columns."""
    for k in (256, 4096):
        a, w = _operands(m, n, k, m + n)
        for dtype in (torch.bfloat16, torch.float32):
            want = plq.ops.fp8_gemm(a, w, out_dtype=dtype, variant=variant)
            _check_product(want, a, w)
            for stride, shift in ((n, 1), (n + 1, 0), (n + 1, 1), (n + 2, 2), (n + 16 - n % 16, 0), (n + 24 - n % 8, 8)):
                store = torch.full((m * stride + shift + 8,), 7.0, dtype=dtype, device="cuda")
                out = store[shift: shift + m * stride].view(m, stride)[:, :n]
                assert torch.equal(plq.ops.fp8_gemm(a, w, out=out, variant=variant), want)
                out[:] = 7.0
                assert torch.all(store == 7.0)
    plq.check_device_status()


def test_rows_do_not_depend_on_each_other(plq):
    """A row or column that is not finite stays alone; a row's result does not depend on the rows around it."""
    for m in (9, 200):
        a, w = _operands(m, 300, 512, 8)
        want = plq.ops.fp8_gemm(a, w)
        a.scales[4, 2] = float("nan")
        got = plq.ops.fp8_gemm(a, w)
        assert torch.all(got[4].isnan())
        keep = torch.arange(m, device="cuda") != 4
        assert torch.equal(got[keep], want[keep])
        w.scales[1, 0] = float("nan")
        got = plq.ops.fp8_gemm(a, w)
        assert torch.all(got[:, 128:256].isnan()) and torch.equal(got[keep][:, :128], want[keep][:, :128]) and torch.equal(got[keep][:, 256:], want[keep][:, 256:])


def test_replayed_in_a_graph_and_on_two_streams(plq):
    x, r, gamma = _rand((3, 1024), 20), _rand((3, 1024), 21), _rand((1024,), 22)
    w = plq.ops.fp8_pack_weight(_rand((5000, 1024), 23, 0.02))

    def step():
        h, p = plq.ops.add_rmsnorm_fp8_pack(x, r, gamma, EPS)
        return plq.ops.fp8_gemm(p, w, out_dtype=torch.float32, static_weights=True)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            y = step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    x.mul_(2.0)
    graph.replay()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(step())
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, y)
    plq.check_device_status()
