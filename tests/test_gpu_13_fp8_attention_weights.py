"""Attention over the E4M3 cache where softmax weights, value blocks and queries of very different size meet: small weights that
are many, blocks whose values dwarf the others', a small query beside a large one.  Each kernel is held to its own rounding."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BLOCK = 64


@pytest.fixture(scope="module")
def plq():
    import plaquant_b200
    from plaquant_b200 import kv_cache  # noqa: F401
    return plaquant_b200


def _cache(plq, batch, n, kv_heads, k, v, k_scale, v_scale):
    """Codes from float values [n, 128] (the same for every sequence and head) and a scale per block."""
    c = plq.kv_cache.Fp8Cache.empty(batch, n, kv_heads, "cuda")
    for codes, scale, x, s in ((c.k, c.k_scale, k, k_scale), (c.v, c.v_scale, v, v_scale)):
        codes.copy_(x.to(torch.float8_e4m3fn).view(torch.uint8)[None, :, None].expand_as(codes))
        scale.copy_(s.expand_as(scale))
    return c


# Rounding of a weight, and what all fixed steps of a block of 64 positions add up to, of the block's own largest weight:
#   f16 (2^-11), then E4M3 + E4M3: half of 2^-3, of that rest half of 2^-3, 2^-9 in all
#   no step is below 2^-9: 64 halves of it are 2^-4, and the block's largest is 2^8 ("few": up to 16 rows per key head), or above 2^7
#   ("many"): 2^-12 or 2^-11 of it
ROUND = {"few": (2.0 ** -9 + 2.0 ** -11, 2.0 ** -12), "many": (2.0 ** -9 + 2.0 ** -11, 2.0 ** -11)}


def _check(out, q, cache, pos, scale=128 ** -0.5):
    """Element by element against float64; a query's elements at or above 2^-9 of its largest are exact, the others off by 2^-17 of
    that at most; a score's float32 arithmetic and exponential by 2^-21 of its size; the result's rounding 2^-8."""
    b, t, heads, _ = q.shape
    group, n = heads // cache.kv_heads, pos + t
    rounding, own = ROUND["few" if t * group <= 16 else "many"]
    for i in range(b):
        s = lambda x: x[i].double().repeat_interleave(BLOCK, -1)[:, :n, None]        # noqa: E731
        k = cache.k[i, :n].contiguous().view(torch.float8_e4m3fn).double().transpose(0, 1) * s(cache.k_scale)
        v = cache.v[i, :n].contiguous().view(torch.float8_e4m3fn).double().transpose(0, 1) * s(cache.v_scale)
        qq = q[i].double().view(t, cache.kv_heads, group, 128).permute(1, 2, 0, 3).reshape(cache.kv_heads, group * t, 128)
        score = qq @ k.transpose(-1, -2) * scale
        seen = (torch.arange(n, device=q.device)[None, :] <= pos + torch.arange(t, device=q.device)[:, None]).repeat(group, 1)
        w = torch.exp(score - score.masked_fill(~seen, -math.inf).amax(-1, keepdim=True)).masked_fill(~seen, 0.0)
        total = w.sum(-1, keepdim=True)
        want = w @ v / total
        blocks = lambda x, d: torch.nn.functional.pad(x, (0, 0, 0, -n % BLOCK) if d == 1 else (0, -n % BLOCK)).unflatten(d, (-1, BLOCK)).amax(d + 1)      # noqa: E731
        top, vmax = blocks(w, 2), blocks(v.abs(), 1)                                  # [kv, rows, blocks], [kv, blocks, 128]
        q_top = qq.abs().amax(-1, keepdim=True)
        dq = torch.where(qq.abs() < 2.0 ** -9 * q_top, torch.minimum(qq.abs(), 2.0 ** -17 * q_top), torch.zeros_like(qq))
        off = w * torch.expm1(abs(scale) * (dq @ k.abs().transpose(-1, -2)) + 2.0 ** -21 * (1 + score.abs()))
        bound = want.abs() * (2.0 ** -8 + off.sum(-1, keepdim=True) / total)
        bound = bound + ((rounding * w + off) @ v.abs() + own * top @ vmax) / total
        put = lambda x: x.view(cache.kv_heads, group, t, 128).permute(2, 0, 1, 3).reshape(t, heads, 128)      # noqa: E731
        err, bound = (out[i].double() - put(want)).abs(), put(bound) * (1 + 2.0 ** -6) + 1e-37
        assert torch.all(err <= bound), (i, float((err / bound).max()))


# rows per key head: 1, 16 (the kernel for few), 32 in runs and whole, a prompt's chunk
SHAPES = [(1, 1, 1, 1), (1, 4, 4, 1), (1, 8, 4, 1), (12, 200, 8, 1), (3, 9, 8, 2)]


@pytest.mark.parametrize("b,t,heads,kv_heads", SHAPES)
@pytest.mark.parametrize("nats", [6.0, 12.0, 13.0, 14.0, 18.0])
def test_a_long_flat_tail_behind_a_first_token(plq, b, t, heads, kv_heads, nats):
    """One position far above a tail of equal scores and equal values: the tail's part of the sum is the result.  Its weights may be
    off by 2^-9 + 2^-11 each, all in the same direction; the 63 that share a block with the first may be lost beside it."""
    n = 131072 if b == 1 else 16384
    k, v = torch.zeros(n, 128, device="cuda"), torch.ones(n, 128, device="cuda")
    k[0], v[0] = 1.0, 0.0
    one = torch.ones(-(-n // BLOCK), device="cuda")
    cache = _cache(plq, b, n, kv_heads, k, v, one, one * 0.5)
    q = torch.full((b, t, heads, 128), nats / 128 ** 0.5, device="cuda").to(torch.bfloat16)
    out = plq.ops.fp8_cache_attention(q, cache, n - t)
    above = math.exp(float(q[0, 0, 0, 0]) * 128 ** 0.5)
    tail = torch.arange(n - t, n, device="cuda", dtype=torch.float64)[None, :, None, None]       # positions behind the first that a query sees
    want = 0.5 * tail / (tail + above)
    # a weight 2^-9 + 2^-11, the steps of a block 2^-11, the result's rounding 2^-8, the exponential of 18
    assert float(((out.double() - want) / want).abs().max()) <= 2.0 ** -8 + 2.0 ** -9 + 2.0 ** -10 + 2.0 ** -16 + 63 / (n - t)
    plq.check_device_status()


@pytest.mark.parametrize("b,t,heads,kv_heads", SHAPES)
@pytest.mark.parametrize("large", [[0], [100], [1, 63, 64, 130], list(range(0, 140, 3))])
@pytest.mark.parametrize("power", [8, 14, 20])
def test_a_channel_of_large_values_takes_nothing_from_the_others(plq, b, t, heads, kv_heads, large, power):
    """Blocks with one strong channel have a larger scale; what the other channels get from the other blocks stays."""
    n = 64 * 150 - 7
    g = torch.Generator(device="cuda").manual_seed(power)
    v = torch.ones(n, 128, device="cuda")
    v_scale = torch.ones(150, device="cuda")
    for j in large:
        v_scale[j] = 2.0 ** power
        v[64 * j: 64 * j + 64] = 0.0
        v[64 * j: 64 * j + 64, 5] = 1.0
    k = torch.randn(n, 128, generator=g, device="cuda")
    cache = _cache(plq, b, n, kv_heads, k, v, torch.ones(150, device="cuda"), v_scale)
    q = (torch.randn(b, t, heads, 128, generator=g, device="cuda") * 0.02).to(torch.bfloat16)
    out = plq.ops.fp8_cache_attention(q, cache, n - t).double()
    _check(out, q, cache, n - t)
    # the other channels are the sum of the weights of the other blocks: 0 .. 1, and no element of theirs is large
    kk = cache.k[0, :, 0].contiguous().view(torch.float8_e4m3fn).double()
    score = (q[0].double() @ kk.t()) * 128 ** -0.5
    seen = torch.arange(n, device="cuda") <= n - t + torch.arange(t, device="cuda")[:, None, None]
    w = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
    want = (w * (v[:, 0] != 0)).sum(-1)
    err = (out[0][..., [0, 4, 6, 127]] / want[..., None] - 1).abs().max()
    assert float(err) <= 2.0 ** -8 + 2.0 ** -9 + 2.0 ** -10 + 2.0 ** -19 * (1 + float(score.abs().max()))
    plq.check_device_status()


@pytest.mark.parametrize("rows", [(1, 1, 1), (2, 8, 1), (1, 16, 2)])
def test_two_value_blocks_of_a_tile_keep_their_own_weights(plq, rows):
    """The second half of a tile of 128 positions: weights of 2^-18.8 of the first half's, values 2^19 times as large."""
    t, heads, kv_heads = rows
    n = 128 + t
    k, v = torch.zeros(n, 128, device="cuda"), torch.zeros(n, 128, device="cuda")
    k[:64] = 1.0
    v[:64, ::2], v[64:, 1::2] = 1.0, 1.0
    v_scale = torch.tensor([1.0, 2.0 ** 19, 2.0 ** 19], device="cuda")[: -(-n // BLOCK)]
    cache = _cache(plq, 1, n, kv_heads, k, v, torch.ones_like(v_scale), v_scale)
    q = torch.full((1, t, heads, 128), 13.0 / 128 ** 0.5, device="cuda").to(torch.bfloat16)
    out = plq.ops.fp8_cache_attention(q, cache, n - t)
    _check(out, q, cache, n - t)
    small = math.exp(-float(q[0, 0, 0, 0]) * 128 ** 0.5)
    behind = 65.0 + torch.arange(t, device="cuda", dtype=torch.float64)[:, None]
    want = behind * small / (64 + behind * small) * 2.0 ** 19
    # a weight 2^-9 + 2^-11, steps 2^-12, the result 2^-8, the exponential of 13
    assert float((out[0, ..., 1].double() / want - 1).abs().max()) <= 2.0 ** -8 + 2.0 ** -9 + 2.0 ** -11 + 2.0 ** -12 + 2.0 ** -17


@pytest.mark.parametrize("t,heads,kv_heads", [(1, 4, 1), (2, 8, 1), (4, 8, 1), (40, 4, 1)])
@pytest.mark.parametrize("power", [10, 20, 40])
def test_a_small_query_beside_a_large_one(plq, t, heads, kv_heads, power):
    """Heads of one group whose queries differ by powers of two: each has its own scale."""
    n, g = 700, torch.Generator(device="cuda").manual_seed(power)
    k = torch.randn(n, 128, generator=g, device="cuda")
    v = torch.randn(n, 128, generator=g, device="cuda")
    k[:, :64] *= 2.0 ** -6                             # what the large query looks at
    k_scale = torch.full((11,), 2.0 ** (power - 6), device="cuda")
    cache = _cache(plq, 1, n, kv_heads, k, v, k_scale, torch.ones(11, device="cuda"))
    q = torch.randn(1, t, heads, 128, generator=g, device="cuda") * 2.0 ** (6 - power)
    q[:, :, 0] = 0.0
    q[:, :, 0, 3] = 2.0 ** 6
    q[:, :, 1:, :64] = 0.0
    q = q.to(torch.bfloat16)
    cache.k.view(n, 128)[:, 3] = 0                     # nothing: its row is the plain mean
    out = plq.ops.fp8_cache_attention(q, cache, n - t)
    _check(out, q, cache, n - t)


@pytest.mark.parametrize("b,t,heads,kv_heads,n", [(1, 1, 8, 1, 3000), (2, 2, 8, 2, 900), (1, 8, 4, 1, 9000), (4, 70, 16, 4, 1500), (2, 300, 8, 2, 300)])
@pytest.mark.parametrize("gain", [1.0, 4.0, 12.0])
def test_scores_and_values_of_every_size(plq, b, t, heads, kv_heads, n, gain):
    """Random blocks whose keys and values differ by powers of two, wide and narrow score distributions."""
    g = torch.Generator(device="cuda").manual_seed(int(gain) + n)
    blocks = -(-n // BLOCK)
    k, v = (torch.randn(n, 128, generator=g, device="cuda") for _ in range(2))
    k_scale, v_scale = (torch.exp2(torch.randint(lo, hi, (blocks,), generator=g, device="cuda").float()) for lo, hi in ((-4, 1), (-6, 7)))
    cache = _cache(plq, b, n, kv_heads, k, v, k_scale, v_scale)
    q = (torch.randn(b, t, heads, 128, generator=g, device="cuda") * gain).to(torch.bfloat16)
    _check(plq.ops.fp8_cache_attention(q, cache, n - t), q, cache, n - t)
    at = torch.full((b,), n - t, device="cuda")
    _check(plq.ops.fp8_cache_attention(q, cache, at), q, cache, n - t)
    plq.check_device_status()


def test_blocks_of_zeros_leave_the_others(plq):
    """Zeros have the smallest scale there is: positions of nothing in front of, between and behind others."""
    for t, heads in ((1, 4), (40, 4)):
        n = 64 * 20
        g = torch.Generator(device="cuda").manual_seed(3)
        k, v = (torch.randn(n, 128, generator=g, device="cuda") for _ in range(2))
        v_scale = torch.full((20,), 2.0 ** -6, device="cuda")
        for j in (0, 1, 5, 6, 12, 19):
            v[64 * j: 64 * j + 64] = 0.0
            v_scale[j] = 2.0 ** -100
        cache = _cache(plq, 1, n, 1, k, v, torch.ones(20, device="cuda"), v_scale)
        q = torch.randn(1, t, heads, 128, generator=g, device="cuda").to(torch.bfloat16)
        _check(plq.ops.fp8_cache_attention(q, cache, n - t), q, cache, n - t)
        cache.v.zero_()
        cache.v_scale.fill_(2.0 ** -100)
        assert torch.all(plq.ops.fp8_cache_attention(q, cache, n - t) == 0)


@pytest.mark.parametrize("b,t,heads,kv_heads,n", [(1, 9, 8, 2, 9000), (1, 64, 32, 8, 8000), (3, 40, 10, 2, 5000), (2, 1, 16, 2, 5000), (1, 4, 16, 4, 3000)])
def test_a_workspace_needs_no_more_than_sixteen_bytes_of_alignment(plq, b, t, heads, kv_heads, n):
    """Workspaces at 0 and at 16 behind a multiple of 32: the same result, and nothing outside them is written."""
    from plaquant_b200 import _lib
    g = torch.Generator(device="cuda").manual_seed(n)
    cache = _cache(plq, b, n, kv_heads, torch.randn(n, 128, generator=g, device="cuda"), torch.randn(n, 128, generator=g, device="cuda"),
                   torch.ones(-(-n // BLOCK), device="cuda"), torch.ones(-(-n // BLOCK), device="cuda"))
    q = torch.randn(b, t, heads, 128, generator=g, device="cuda").to(torch.bfloat16)
    want = plq.ops.fp8_cache_attention(q, cache, n - t)
    lib, status = _lib.lib(), plq.ops.status_word("cuda")
    need = lib.plq_fp8_attention_workspace_bytes(b, t, heads, kv_heads, n)
    assert need > 0
    for shift in (0, 16):
        room = torch.full((need + 128,), 0xA5, dtype=torch.uint8, device="cuda")
        at = (room.data_ptr() + 63) // 32 * 32 + shift
        out = torch.empty_like(q)
        st = lib.plq_fp8_attention(q.data_ptr(), cache.k.data_ptr(), cache.k_scale.data_ptr(), cache.v.data_ptr(), cache.v_scale.data_ptr(), b, t, heads,
                                   kv_heads, n, None, 0, n - t, n, 128 ** -0.5, out.data_ptr(), at, need, status.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert st == 0
        torch.cuda.synchronize()
        first = at - room.data_ptr()
        assert torch.equal(out, want) and torch.all(room[:first] == 0xA5) and torch.all(room[first + need:] == 0xA5)
    plq.check_device_status()


@pytest.mark.parametrize("t,heads,kv_heads,n", [(1, 4, 1, 300), (1, 8, 2, 5000), (4, 4, 1, 700), (40, 4, 2, 300), (40, 8, 2, 5000), (300, 2, 2, 300)])
@pytest.mark.parametrize("scale", [1e3, 1e6, 1e8, -1e8, 1e12, 1e25])
def test_scores_beyond_what_float32_counts(plq, t, heads, kv_heads, n, scale):
    """Scores so large that their differences are millions: the largest one's value is the result, wherever it is well apart (a
    score is off by 2^-21 of its size, and differences count in units of that: 2^-14 of it are 128)."""
    g = torch.Generator(device="cuda").manual_seed(n + t)
    k, v = (torch.randn(n, 128, generator=g, device="cuda") for _ in range(2))
    cache = _cache(plq, 2, n, kv_heads, k, v, torch.full((-(-n // BLOCK),), 0.5, device="cuda"), torch.ones(-(-n // BLOCK), device="cuda"))
    q = torch.randn(2, t, heads, 128, generator=g, device="cuda").to(torch.bfloat16)
    kk, vv = (x.view(torch.float8_e4m3fn).double() for x in (cache.k[0, :, 0], cache.v[0, :, 0]))
    score = (q.double() @ kk.t()) * 0.5 * scale
    score = score.masked_fill(torch.arange(n, device="cuda") > n - t + torch.arange(t, device="cuda")[:, None, None], -math.inf)
    best, at = score.topk(2, -1)
    size = score.masked_fill(score == -math.inf, 0.0).abs().amax(-1)
    clear = (best[..., 0] - best[..., 1] > 2.0 ** -14 * size + 30.0) & (at[..., 0] >= 0)
    assert clear.double().mean() > 0.9
    out = plq.ops.fp8_cache_attention(q, cache, n - t, scale=scale).double()
    want = vv[at[..., 0]]
    # the weight 2^-9 + 2^-11, the result 2^-8; what is left of the others e^-30 each
    err = (out - want).abs() - want.abs() * (2.0 ** -8 + 2.0 ** -9 + 2.0 ** -11) - 1e-8
    assert out.isfinite().all() and float(err[clear].max()) <= 0
    plq.check_device_status()
