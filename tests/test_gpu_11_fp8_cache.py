"""The E4M3 key / value cache: append (RoPE, block scales, growth of a block's scale) to the last bit against a restatement of
its definition, attention against float64."""
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


def _cache(plq, batch, room, kv_heads, seed=0):
    """A cache whose unwritten positions hold anything: random bytes (NaN codes among them) and scales."""
    g = torch.Generator().manual_seed(seed)
    c = plq.kv_cache.Fp8Cache.empty(batch, room, kv_heads, "cuda")
    for codes, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
        codes.copy_(torch.randint(0, 256, codes.shape, generator=g, dtype=torch.uint8))
        scale.copy_(torch.randn(scale.shape, generator=g))
        scale.view(-1)[::3] = float("nan")
    return c


def _clone(plq, c):
    return plq.kv_cache.Fp8Cache(c.k.clone(), c.k_scale.clone(), c.v.clone(), c.v_scale.clone())


def _same(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip((a.k, a.k_scale, a.v, a.v_scale), (b.k, b.k_scale, b.v, b.v_scale)))


def _angles(positions):
    inv = 1.0 / (500000.0 ** (torch.arange(0, 128, 2, dtype=torch.float64) / 128))
    ang = positions.double().cpu()[..., None] * inv
    ang = torch.cat([ang, ang], -1)
    return ang.cos().float().cuda().contiguous(), ang.sin().float().cuda().contiguous()


def _rope(x, cos, sin):
    """x * cos + rotate_half(x) * sin, every float32 operation rounded on its own, one rounding to bf16."""
    f = x.float()
    return (f * cos + torch.cat([-f[..., 64:], f[..., :64]], -1) * sin).to(torch.bfloat16)


def _scale_of(amax):
    """The smallest 2^e >= amax / 448 with e >= -100."""
    m, e = math.frexp(amax)
    return 2.0 ** max(e - (9 if m <= 0.875 else 8), -100) if amax > 0 else 2.0 ** -100


def _append_side(codes, scales, new, pos):
    """One sequence: new [t, kv_heads, 128] bf16 into codes [room, kv_heads, 128], scales [kv_heads, blocks], on the CPU."""
    t = new.shape[0]
    for block in range(pos // BLOCK, (pos + t - 1) // BLOCK + 1):
        lo, hi = block * BLOCK, min(block * BLOCK + BLOCK, pos + t)
        start = max(lo, pos)
        for h in range(new.shape[1]):
            x = new[start - pos:hi - pos, h].float()
            old = float(scales[h, block]) if start > lo else 0.0
            if not (torch.isfinite(x).all() and old == old):
                scales[h, block] = float("nan")
                codes[start:hi, h] = 0
                continue
            s = max(_scale_of(float(x.abs().max())), old)
            if start > lo and s != old:
                was = codes[lo:start, h].contiguous().view(torch.float8_e4m3fn).float()
                codes[lo:start, h] = (was * (old / s)).to(torch.float8_e4m3fn).view(torch.uint8)
            codes[start:hi, h] = (x / torch.tensor(s)).to(torch.float8_e4m3fn).view(torch.uint8)
            scales[h, block] = s


def _append(plq, cache, qkv, cos, sin, heads, kv_heads, pos):
    """The definition, in place on a CPU copy; returns (rotated queries, cache on the GPU)."""
    b, t, _ = qkv.shape
    x = qkv.view(b, t, -1, 128)
    cos, sin = cos.view(-1, t, 1, 128), sin.view(-1, t, 1, 128)
    k, v = _rope(x[:, :, heads:heads + kv_heads], cos, sin).cpu(), x[:, :, heads + kv_heads:].cpu()
    side = [[c.cpu(), s.cpu()] for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
    for i in range(b):
        if pos[i] < 0:
            continue
        for (codes, scales), new in zip(side, (k, v)):
            _append_side(codes[i], scales[i], new[i], pos[i])
    return _rope(x[:, :, :heads], cos, sin), plq.kv_cache.Fp8Cache(*(x.cuda() for s in side for x in s))


def _qkv(b, t, heads, kv_heads, seed, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, t, (heads + 2 * kv_heads), 128, generator=g) * gain
    x[..., ::29] *= 6.0
    x *= torch.exp2(torch.randint(-3, 4, (b, t, 1, 1), generator=g).float())          # rows of different size: scales that grow
    return x.flatten(2).to(torch.bfloat16).cuda()


@pytest.mark.parametrize("b,t,heads,kv_heads,pos", [
    (1, 1, 1, 1, [0]), (1, 1, 4, 1, [63]), (2, 1, 8, 2, [64, 64]), (3, 5, 2, 2, [60, 60, 60]), (1, 64, 4, 4, [0]), (1, 65, 4, 2, [0]),
    (2, 200, 8, 4, [37, 37]), (1, 700, 4, 1, [130]),
    (3, 1, 8, 8, [0, 5, 127]), (4, 3, 4, 2, [61, 0, 126, 199]), (3, 130, 6, 3, [1, 63, 64]), (3, 2, 4, 2, [-1, 7, -5])])
@pytest.mark.parametrize("where", ["host", "device"])
def test_append_bit_exact(plq, b, t, heads, kv_heads, pos, where):
    same = len(set(pos)) == 1
    if where == "host" and not same:
        pytest.skip("sequences at different positions are given in device memory")
    room = max(max(pos), 0) + t + 3
    cache = _cache(plq, b, room, kv_heads, 1)
    for step in range(3):                              # from an empty cache, and behind what the calls before left
        start = [p if p < 0 else (0 if step == 0 else p) for p in pos]
        n = t if step else max(max(pos), 1)             # the first call fills up to the largest position
        qkv = _qkv(b, n, heads, kv_heads, 10 + step, gain=(1.0, 2.0, 0.5)[step])
        at = torch.tensor(start)[:, None] + torch.arange(n)
        cos, sin = _angles(at if not same else at[0])
        want_q, want = _append(plq, cache, qkv, cos, sin, heads, kv_heads, start)
        p = start[0] if where == "host" else torch.tensor(start if not same or b == 1 else start[:1], dtype=torch.int64, device="cuda")
        q = plq.ops.rope_kv_append_fp8(qkv, cos, sin, heads, kv_heads, cache, p)
        assert torch.equal(q, want_q)
        assert _same(cache, want)
    plq.check_device_status()


def test_append_token_by_token_with_growing_values(plq):
    """Every token larger than the one before: the block's scale moves with almost every call."""
    heads, kv_heads = 2, 2
    cache = _cache(plq, 1, 130, kv_heads, 2)
    for i in range(130):
        qkv = _qkv(1, 1, heads, kv_heads, 100 + i, gain=2.0 ** (i % 64 - 20))
        cos, sin = _angles(torch.tensor([i]))
        _, want = _append(plq, cache, qkv, cos, sin, heads, kv_heads, [i])
        plq.ops.rope_kv_append_fp8(qkv, cos, sin, heads, kv_heads, cache, i)
        assert _same(cache, want)


def test_append_values_at_the_border_of_a_scale(plq):
    """448, 2^-100 * 448, zeros, the largest and the smallest bf16, not finite ones."""
    for i, v in enumerate([448.0, 450.0, 447.0, 0.0, 3.38e38, 1e-38, 2.0 ** -100 * 448, 2.0 ** -91, -448.0, float("inf"), float("-inf"), float("nan")]):
        cache = _cache(plq, 1, 70, 1, 3)
        qkv = torch.zeros(1, 66, 3 * 128, dtype=torch.bfloat16, device="cuda")
        qkv[0, 3, 128 + 17] = v
        qkv[0, 5, 256 + 100] = v
        qkv[0, 7, 256:] = 1.0
        cos, sin = torch.ones(66, 128, device="cuda"), torch.zeros(66, 128, device="cuda")
        _, want = _append(plq, cache, qkv, cos, sin, 1, 1, [0])
        plq.ops.rope_kv_append_fp8(qkv, cos, sin, 1, 1, cache, 0)
        if v == v and abs(v) < 1e39:
            assert _same(cache, want), v
        else:
            assert cache.v_scale[0, 0, 0].isnan() and not cache.v_scale[0, 0, 1].isnan()
            assert torch.all(cache.v[0, :64] == 0)


def test_append_refuses_what_does_not_fit(plq):
    heads, kv_heads = 4, 2
    cache = _cache(plq, 2, 100, kv_heads, 4)
    qkv = _qkv(2, 3, heads, kv_heads, 5)
    cos, sin = _angles(torch.arange(3))
    before = _clone(plq, cache)
    with pytest.raises(plq.PlqError):
        plq.ops.rope_kv_append_fp8(qkv, cos, sin, heads, kv_heads, cache, 98)
    plq.ops.rope_kv_append_fp8(qkv, cos, sin, heads, kv_heads, cache, torch.tensor([98, -1], device="cuda"))
    assert _same(cache, before)
    with pytest.raises(plq.PlqError):
        plq.check_device_status()
    plq.check_device_status()


# ---- attention -------------------------------------------------------------------------------------------------------
def _filled(plq, batch, room, kv_heads, lengths, seed, gain=1.0):
    """A cache filled by the append itself, `lengths` positions of every sequence, anything behind them."""
    cache = _cache(plq, batch, room, kv_heads, seed)
    n = max(lengths)
    if n > 0:
        g = torch.Generator(device="cuda").manual_seed(seed)
        x = torch.randn(batch, n, 3 * kv_heads, 128, generator=g, device="cuda") * gain
        x[..., ::37] *= 4.0
        full = plq.kv_cache.Fp8Cache.empty(batch, n, kv_heads, "cuda")
        ones = torch.ones(n, 128, device="cuda")
        plq.ops.rope_kv_append_fp8(x.flatten(2).to(torch.bfloat16), ones, torch.zeros_like(ones), kv_heads, kv_heads, full, 0)
        for i, m in enumerate(lengths):
            cache.k[i, :m], cache.v[i, :m] = full.k[i, :m], full.v[i, :m]
            blocks = -(-m // BLOCK)
            cache.k_scale[i, :, :blocks], cache.v_scale[i, :, :blocks] = full.k_scale[i, :, :blocks], full.v_scale[i, :, :blocks]
    return cache


def _check_attention(out, q, cache, pos, scale=128 ** -0.5):
    """Against float64, within what the arithmetic allows of either kernel, element by element:
      a weight w is two codes - off by 2^-8 of itself at most (E4M3: half of 2^-3; of that rest, E5M2: half of 2^-2 of at most
      2^-4 = 2^-7 in all against the binade, 2^-8 of its largest value) - or by half a step: 2^-18 of the largest weight of its
      128 positions (E4M3 alone, the largest brought to 256), 2^-16 of the row's largest w vs over its own vs (E4M3 + E5M2,
      the largest at 4 or more: below 2^-6 E4M3 leaves up to 2^-10, of which E5M2 is off by 2^-4, together 2^-14 = 2^-16 of 4);
      a query's element that is below 2^-9 of the row's largest is off by 2^-17 of it or by itself, the others are exact;
      the score's float32 arithmetic and exponential by 2^-21 of its size; the result's rounding by 2^-8."""
    b, t, heads, _ = q.shape
    group = heads // cache.kv_heads
    for i in range(b):
        n = pos[i] + t
        if pos[i] < 0:
            assert torch.all(out[i] == 0)
            continue
        s = lambda x: x[i].double().repeat_interleave(BLOCK, -1)[:, :n, None]        # noqa: E731
        k = cache.k[i, :n].contiguous().view(torch.float8_e4m3fn).double().transpose(0, 1) * s(cache.k_scale)
        v = cache.v[i, :n].contiguous().view(torch.float8_e4m3fn).double().transpose(0, 1) * s(cache.v_scale)
        vs = s(cache.v_scale)[..., 0][:, None]                                                     # [kv, 1, n]
        qq = q[i].double().view(t, cache.kv_heads, group, 128).permute(1, 2, 0, 3).reshape(cache.kv_heads, group * t, 128)
        score = qq @ k.transpose(-1, -2) * scale
        seen = (torch.arange(n, device=q.device)[None, :] <= pos[i] + torch.arange(t, device=q.device)[:, None]).repeat(group, 1)
        w = torch.exp(score - score.masked_fill(~seen, -math.inf).amax(-1, keepdim=True)).masked_fill(~seen, 0.0)
        total = w.sum(-1, keepdim=True)
        want = w @ v / total
        tile = torch.nn.functional.pad(w, (0, -n % 128)).unflatten(-1, (-1, 128)).amax(-1).repeat_interleave(128, -1)[..., :n]
        step = torch.maximum(2.0 ** -18 * tile, 2.0 ** -16 * (w * vs).amax(-1, keepdim=True) / vs)
        top = qq.abs().amax(-1, keepdim=True)
        dq = torch.where(qq.abs() < 2.0 ** -9 * top, torch.minimum(qq.abs(), 2.0 ** -17 * top), torch.zeros_like(qq))
        off = w * (torch.expm1(abs(scale) * (dq @ k.abs().transpose(-1, -2)) + 2.0 ** -21 * (1 + score.abs())))
        err_w = torch.maximum(2.0 ** -8 * w, step) * seen + off
        bound = want.abs() * (2.0 ** -8 + off.sum(-1, keepdim=True) / total) + err_w @ v.abs() / total
        put = lambda x: x.view(cache.kv_heads, group, t, 128).permute(2, 0, 1, 3).reshape(t, heads, 128)      # noqa: E731
        err, bound = (out[i].double() - put(want)).abs(), put(bound) * (1 + 2.0 ** -6) + 1e-37
        assert torch.all(err <= bound), (i, float((err / bound).max()))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 1), (8, 8), (12, 4), (16, 1), (40, 2), (33, 1)])
@pytest.mark.parametrize("t,pos", [(1, 0), (1, 1), (1, 62), (1, 63), (1, 64), (1, 127), (1, 128), (1, 300), (2, 0), (3, 126), (5, 1000), (40, 0), (33, 95)])
def test_attention(plq, heads, kv_heads, t, pos):
    b = 2
    cache = _filled(plq, b, pos + t + 5, kv_heads, [pos + t] * b, heads * 1000 + t + pos)
    q = (_rand_q((b, t, heads, 128), t + pos)).cuda()
    out = plq.ops.fp8_cache_attention(q, cache, pos)
    _check_attention(out, q, cache, [pos] * b)
    at = torch.tensor([pos], device="cuda")
    assert torch.equal(plq.ops.fp8_cache_attention(q, cache, at, ctx=pos + t), out)          # the same split, the same bits
    _check_attention(plq.ops.fp8_cache_attention(q, cache, at), q, cache, [pos] * b)
    plq.check_device_status()


def _rand_q(shape, seed, gain=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * gain).to(torch.bfloat16)


@pytest.mark.parametrize("t", [1, 4, 70])
@pytest.mark.parametrize("lengths", [[1, 500, 64], [0, 129, 2000], [0, 0, 0], [65, 64, 63], [5000, 1, 0]])
def test_attention_of_ragged_batches(plq, t, lengths):
    """Sequences of different lengths, one that sits out."""
    pos = [n if n > 0 else -1 for n in lengths]
    room = max(lengths) + t + 60
    cache = _filled(plq, 3, room, 2, [p + t if p >= 0 else 0 for p in pos], 7)
    q = _rand_q((3, t, 8, 128), 8).cuda()
    out = plq.ops.fp8_cache_attention(q, cache, torch.tensor(pos, device="cuda"))
    _check_attention(out, q, cache, pos)
    plq.check_device_status()


@pytest.mark.parametrize("b,t,heads,kv_heads,pos", [(1, 1, 64, 8, 40000), (1, 2, 8, 1, 70001), (16, 1, 32, 8, 4095), (2, 600, 8, 2, 0), (1, 300, 16, 2, 3000)])
def test_attention_of_ordinary_sizes(plq, b, t, heads, kv_heads, pos):
    cache = _filled(plq, b, pos + t, kv_heads, [pos + t] * b, 9)
    q = _rand_q((b, t, heads, 128), 10).cuda()
    out = plq.ops.fp8_cache_attention(q, cache, pos)
    _check_attention(out, q, cache, [pos] * b)
    assert torch.equal(out, plq.ops.fp8_cache_attention(q, cache, pos))
    plq.check_device_status()


@pytest.mark.parametrize("gain,q_gain,scale", [(1.0, 30.0, None), (1e-3, 1.0, None), (1e4, 1e-4, None), (1.0, 1.0, 0.0), (1.0, 0.0, None), (1.0, 1.0, -0.3), (1e-30, 1e30, None)])
def test_attention_of_sharp_flat_large_and_small_scores(plq, gain, q_gain, scale):
    cache = _filled(plq, 1, 900, 2, [900], 11, gain)
    q = _rand_q((1, 3, 8, 128), 12, q_gain).cuda()
    out = plq.ops.fp8_cache_attention(q, cache, 897, scale=scale)
    _check_attention(out, q, cache, [897], 128 ** -0.5 if scale is None else scale)


def test_attention_where_one_position_outweighs_the_others(plq):
    """A first token with a score far above the rest and next to no value, and a block of large values with low scores."""
    cache = _filled(plq, 1, 1500, 1, [1500], 13)
    q = _rand_q((1, 1, 4, 128), 14).cuda()
    first = plq.kv_cache.Fp8Cache.empty(1, 1500, 1, "cuda")
    row = torch.zeros(1, 1, 3 * 128, dtype=torch.bfloat16, device="cuda")
    row[..., 128:256] = q.float().mean(2).to(torch.bfloat16) * 3
    row[..., 256:] = 1e-3
    one = torch.ones(1, 128, device="cuda")
    plq.ops.rope_kv_append_fp8(row, one, one * 0, 1, 1, first, 0)
    for dst, src in ((cache.k, first.k), (cache.v, first.v)):
        dst[:, 1:64] = 0
        dst[:, 0] = src[:, 0]
    cache.k_scale[..., 0], cache.v_scale[..., 0] = first.k_scale[..., 0], first.v_scale[..., 0]
    cache.v_scale[..., 5] *= 2.0 ** 12
    _check_attention(plq.ops.fp8_cache_attention(q, cache, 1499), q, cache, [1499])


def test_attention_of_equal_values_returns_them(plq):
    """Weights and their sum belong together: a cache of one value gives that value."""
    cache = _filled(plq, 1, 777, 1, [777], 15)
    cache.v.fill_(0x38)                                # 1.0
    cache.v_scale.fill_(0.25)
    q = _rand_q((1, 7, 4, 128), 16).cuda()
    out = plq.ops.fp8_cache_attention(q, cache, 770)
    assert torch.all((out.float() - 0.25).abs() <= 0.25 * (2.0 ** -8 + 2.0 ** -11))


def test_attention_keeps_what_is_not_finite_where_it_is_seen(plq):
    """A block of NaN reaches the rows that see it and no others; a query of NaN or infinity its own row alone."""
    b, t, pos = 1, 100, 150
    for side in ("k_scale", "v_scale"):
        cache = _filled(plq, b, 256, 2, [250], 17)
        q = _rand_q((b, t, 8, 128), 18).cuda()
        want = plq.ops.fp8_cache_attention(q, cache, pos)
        getattr(cache, side)[0, 1, 3] = float("nan")              # positions 192 .. 255 of the second key head
        got = plq.ops.fp8_cache_attention(q, cache, pos)
        hit = torch.zeros(b, t, 8, dtype=torch.bool, device="cuda")
        hit[:, 192 - pos:, 4:] = True
        assert torch.all(got[hit].isnan()) and torch.equal(got[~hit], want[~hit])
    q[0, 7, 3, 5], q[0, 9, 6, 0] = float("nan"), float("inf")
    cache = _filled(plq, b, 256, 2, [250], 17)
    got = plq.ops.fp8_cache_attention(q, cache, pos)
    hit = torch.zeros(b, t, 8, dtype=torch.bool, device="cuda")
    hit[0, 7, 3] = hit[0, 9, 6] = True
    assert torch.all(got[hit].isnan()) and not got[~hit].isnan().any()
    # positions behind the last one may hold NaN codes and scales (every cache here does)
    plq.check_device_status()


# ---- many queries: rows of a tile are queries x heads of a group --------------------------------------------------------
@pytest.mark.parametrize("b,t,heads,kv_heads,pos", [(18, 9, 4, 1, 0), (18, 33, 1, 1, 0), (3, 129, 12, 6, 70), (5, 65, 16, 4, 1000), (2, 256, 9, 9, 127), (9, 64, 8, 2, 64),
                                                    (1, 1000, 40, 8, 0), (2, 300, 16, 2, 5000), (18, 300, 5, 1, 63)])
def test_attention_of_many_queries(plq, b, t, heads, kv_heads, pos):
    cache = _filled(plq, b, pos + t + 5, kv_heads, [pos + t] * b, heads * 100 + t + pos)
    q = _rand_q((b, t, heads, 128), t + pos).cuda()
    out = plq.ops.fp8_cache_attention(q, cache, pos)
    _check_attention(out, q, cache, [pos] * b)
    assert torch.equal(plq.ops.fp8_cache_attention(q, cache, torch.tensor([pos], device="cuda")), out)
    plq.check_device_status()


# ---- more rows than a tile of the split kernel has, behind positions enough for it to be the faster one ------------------
@pytest.mark.parametrize("b,t,heads,kv_heads,pos", [(1, 9, 8, 2, 9000), (2, 33, 4, 4, 5001), (1, 40, 10, 2, 8191)])
def test_several_row_tiles_behind_a_long_past(plq, b, t, heads, kv_heads, pos):
    cache = _filled(plq, b, pos + t + 70, kv_heads, [pos + t] * b, t + pos)
    q = _rand_q((b, t, heads, 128), t + pos).cuda()
    out = plq.ops.fp8_cache_attention(q, cache, pos)
    _check_attention(out, q, cache, [pos] * b)
    at = torch.tensor([pos - 4100 * i for i in range(b)], device="cuda")
    _check_attention(plq.ops.fp8_cache_attention(q, cache, at), q, cache, at.tolist())
    plq.check_device_status()


@pytest.mark.parametrize("t,heads,kv_heads,pos", [(128, 8, 2, [4000]), (24, 32, 4, [9000]), (100, 12, 2, [5000, 130, -1]), (17, 3, 1, [3000, 0, 2047, 511]),
                                                  (65, 16, 1, [20000]), (300, 5, 5, [1, 7000])])
def test_many_queries_in_runs(plq, t, heads, kv_heads, pos):
    """Long pasts and few rows: every sequence cut along its positions; short ones are one run, absent ones none."""
    b, room = len(pos), max(pos) + t + 70
    cache = _filled(plq, b, room, kv_heads, [p + t if p >= 0 else 0 for p in pos], t + heads)
    q = _rand_q((b, t, heads, 128), t).cuda()
    at = torch.tensor(pos, device="cuda")
    out = plq.ops.fp8_cache_attention(q, cache, at)
    _check_attention(out, q, cache, pos)
    assert torch.equal(plq.ops.fp8_cache_attention(q, cache, at, ctx=max(pos) + t), plq.ops.fp8_cache_attention(q, cache, at, ctx=max(pos) + t))
    plq.check_device_status()
    over = torch.tensor([room - t + 1] + pos[1:], device="cuda")
    out = plq.ops.fp8_cache_attention(q, cache, over)
    assert torch.all(out[0] == 0)
    for i in range(1, b):
        _check_attention(out[i: i + 1], q[i: i + 1], plq.kv_cache.Fp8Cache(*(x[i: i + 1] for x in (cache.k, cache.k_scale, cache.v, cache.v_scale))), pos[i: i + 1])
    with pytest.raises(plq.PlqError):
        plq.check_device_status()


@pytest.mark.parametrize("lengths", [[0, 129, 500, -1, 63, 64], [1000, 2, 1, 190, -1, 0]])
def test_many_queries_of_ragged_batches(plq, lengths):
    pos = [n - 1 if n == 0 else n for n in lengths]
    cache = _filled(plq, 6, max(lengths) + 160, 3, [p + 100 if p >= 0 else 0 for p in pos], 50)
    q = _rand_q((6, 100, 6, 128), 51).cuda()
    _check_attention(plq.ops.fp8_cache_attention(q, cache, torch.tensor(pos, device="cuda")), q, cache, pos)
    q = _rand_q((6, 100, 6, 128), 51).cuda()
    over = torch.tensor([max(lengths) + 61] + pos[1:], device="cuda")
    out = plq.ops.fp8_cache_attention(q, cache, over)
    assert torch.all(out[0] == 0)
    with pytest.raises(plq.PlqError):
        plq.check_device_status()


@pytest.mark.parametrize("gain,q_gain,scale", [(1.0, 30.0, None), (1e-3, 1.0, None), (1e4, 1e-4, None), (1.0, 1.0, 0.0), (1.0, 0.0, None), (1.0, 1.0, -0.3), (1e-30, 1e30, None)])
def test_many_queries_of_sharp_flat_large_and_small_scores(plq, gain, q_gain, scale):
    cache = _filled(plq, 5, 900, 4, [900] * 5, 52, gain)
    q = _rand_q((5, 70, 16, 128), 53, q_gain).cuda()
    out = plq.ops.fp8_cache_attention(q, cache, 830, scale=scale)
    _check_attention(out, q, cache, [830] * 5, 128 ** -0.5 if scale is None else scale)


def test_many_queries_where_the_maximum_moves(plq):
    """Keys that grow along the cache: every tile's scores exceed those before, and then fall again; blocks of V of very
    different size, the largest where nobody looks."""
    cache = _filled(plq, 5, 1500, 4, [1500] * 5, 54)
    ramp = torch.cat([torch.arange(12), torch.arange(12).flip(0)])[: cache.k_scale.shape[-1]]
    cache.k_scale.mul_(torch.exp2((ramp - 8).float()).cuda())
    q = _rand_q((5, 200, 16, 128), 55, 1.0).cuda()
    _check_attention(plq.ops.fp8_cache_attention(q, cache, 1300), q, cache, [1300] * 5)
    cache.v_scale[..., ::3] *= 2.0 ** -9
    cache.k_scale[..., 1::3] *= 2.0 ** -12
    _check_attention(plq.ops.fp8_cache_attention(q, cache, 1300), q, cache, [1300] * 5)


def test_many_queries_keep_what_is_not_finite_where_it_is_seen(plq):
    b, t, pos = 9, 100, 150
    for side in ("k_scale", "v_scale"):
        cache = _filled(plq, b, 256, 2, [250] * b, 56)
        q = _rand_q((b, t, 8, 128), 57).cuda()
        want = plq.ops.fp8_cache_attention(q, cache, pos)
        getattr(cache, side)[1, 1, 3] = float("nan")              # positions 192 .. 255 of a sequence's second key head
        got = plq.ops.fp8_cache_attention(q, cache, pos)
        hit = torch.zeros(b, t, 8, dtype=torch.bool, device="cuda")
        hit[1, 192 - pos:, 4:] = True
        assert torch.all(got[hit].isnan()) and torch.equal(got[~hit], want[~hit])
    cache = _filled(plq, b, 256, 2, [250] * b, 56)
    q[0, 7, 3, 5], q[8, 9, 6, 0] = float("nan"), float("inf")
    got = plq.ops.fp8_cache_attention(q, cache, pos)
    hit = torch.zeros(b, t, 8, dtype=torch.bool, device="cuda")
    hit[0, 7, 3] = hit[8, 9, 6] = True
    assert torch.all(got[hit].isnan()) and torch.equal(got[~hit], want[~hit])


def test_attention_reports_positions_outside_the_cache(plq):
    cache = _filled(plq, 2, 100, 1, [100, 100], 19)
    q = _rand_q((2, 2, 4, 128), 20).cuda()
    with pytest.raises(plq.PlqError):
        plq.ops.fp8_cache_attention(q, cache, 99)
    out = plq.ops.fp8_cache_attention(q, cache, torch.tensor([99, 98], device="cuda"))
    assert torch.all(out[0] == 0)
    _check_attention(out[1:], q[1:], plq.kv_cache.Fp8Cache(cache.k[1:], cache.k_scale[1:], cache.v[1:], cache.v_scale[1:]), [98])
    with pytest.raises(plq.PlqError):
        plq.check_device_status()


def test_nobody_attends(plq):
    """A negative position given by the host, no queries, no sequences; split over the device or not."""
    cache = _filled(plq, 3, 3000, 2, [3000] * 3, 60)
    for t in (1, 40, 300):
        assert torch.all(plq.ops.fp8_cache_attention(_rand_q((3, t, 8, 128), 61).cuda(), cache, -1) == 0)
    before = _clone(plq, cache)
    qkv, one = _qkv(3, 2, 8, 2, 62), torch.ones(2, 128, device="cuda")
    plq.ops.rope_kv_append_fp8(qkv, one, one * 0, 8, 2, cache, -3)
    assert _same(before, cache)
    assert plq.ops.fp8_cache_attention(torch.empty(3, 0, 8, 128, dtype=torch.bfloat16, device="cuda"), cache, 5).shape == (3, 0, 8, 128)
    none = plq.kv_cache.Fp8Cache.empty(0, 64, 2, "cuda")
    assert plq.ops.fp8_cache_attention(torch.empty(0, 1, 8, 128, dtype=torch.bfloat16, device="cuda"), none, 5).shape == (0, 1, 8, 128)
    plq.check_device_status()


def test_refusals_on_the_device(plq):
    cache = _filled(plq, 2, 100, 2, [100, 100], 63)
    q = _rand_q((2, 1, 8, 128), 64).cuda()
    attend = plq.ops.fp8_cache_attention
    for bad in (q[:, :, :7], q.float(), q.transpose(1, 2), q[..., :64], q[:1]):
        with pytest.raises((TypeError, ValueError)):
            attend(bad, cache, 5)
    for pos in (torch.tensor([1, 2, 3], device="cuda"), torch.tensor([1], dtype=torch.int32, device="cuda"), torch.tensor([1, 2])):
        with pytest.raises(TypeError):
            attend(q, cache, pos)
    with pytest.raises(plq.PlqError):
        attend(q, cache, torch.tensor([1], device="cuda"), ctx=101)
    qkv, one = _qkv(2, 1, 8, 2, 65), torch.ones(1, 128, device="cuda")
    with pytest.raises(TypeError):
        plq.ops.rope_kv_append_fp8(qkv, one, torch.ones(2, 128, device="cuda"), 8, 2, cache, 0)
    with pytest.raises(TypeError):
        plq.ops.rope_kv_append_fp8(qkv[:, :, :-128], one, one, 8, 2, cache, 0)
    with pytest.raises(TypeError):
        plq.ops.rope_kv_append_fp8(qkv, one, one, 10, 1, cache, 0)
    g = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    x = torch.ones(2, 512, dtype=torch.bfloat16, device="cuda")
    for bad in (dict(gamma=g[:256]), dict(gamma=g.float())):
        with pytest.raises(TypeError):
            plq.ops.fp8_pack(x, **bad)
    with pytest.raises(TypeError):
        plq.ops.add_rmsnorm_fp8_pack(x, x, None, 1e-6)
    with pytest.raises(plq.PlqError):
        plq.ops.fp8_pack(x[:, :40].contiguous())
    a, w = plq.ops.fp8_pack(x), plq.ops.fp8_pack_weight(x)
    for bad in ((w, w), (a, a), (plq.ops.fp8_pack(x[:, :256]), w)):
        with pytest.raises(ValueError):
            plq.ops.fp8_gemm(*bad)
    with pytest.raises(TypeError):
        plq.ops.fp8_gemm(plq.ops.Fp8Matrix(a.codes, a.scales[:, :2], 1), w)
    with pytest.raises(TypeError):
        plq.ops.fp8_gemm(a, w, out_dtype=torch.float16)
    for out in (torch.empty(2, 3, device="cuda"), torch.empty(3, 2, device="cuda"), torch.empty(2, 4, device="cuda")[:, ::2], torch.empty(1, 2, device="cuda").expand(2, 2)):
        with pytest.raises(RuntimeError):
            plq.ops.fp8_gemm(a, w, out=out)


def test_step_in_a_graph_at_moving_positions(plq):
    """Append and attention captured once, replayed while the position in device memory moves; two graphs of different shapes
    and an eager stream beside them."""
    heads, kv_heads, b, room = 8, 2, 3, 700
    eager, caught = _filled(plq, b, room, kv_heads, [600] * b, 21), None
    caught = _clone(plq, eager)
    pos = torch.tensor([500, 70, -1], device="cuda")
    qkv = _qkv(b, 1, heads, kv_heads, 22)
    cos, sin = torch.ones(1, 128, device="cuda"), torch.zeros(1, 128, device="cuda")

    def step(cache):
        q = plq.ops.rope_kv_append_fp8(qkv, cos, sin, heads, kv_heads, cache, pos)
        return plq.ops.fp8_cache_attention(q, cache, pos)
    step(_clone(plq, eager))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        step(_clone(plq, eager))
        side.synchronize()
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                y = step(caught)
            graphs.append((g, y))
    torch.cuda.synchronize()
    for i in range(6):
        qkv.copy_(_qkv(b, 1, heads, kv_heads, 30 + i))
        g, y = graphs[i % 2]
        g.replay()
        want = step(eager)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and _same(eager, caught)
        pos.add_((pos >= 0).long())
    plq.check_device_status()


def test_long_cache_behind_the_32_bit_border(plq):
    """More than 2^32 bytes of codes: the last sequence's rows and scales are found."""
    b, kv_heads, room = 5, 8, (1 << 32) // (4 * 8 * 128) + 64
    cache = plq.kv_cache.Fp8Cache.empty(b, room, kv_heads, "cuda")
    for x in (cache.k, cache.v):
        x.zero_()
    for x in (cache.k_scale, cache.v_scale):
        x.fill_(2.0 ** -8)
    pos = torch.tensor([3, -1, room - 700, -1, room - 300], device="cuda")
    qkv = _qkv(b, 300, 16, kv_heads, 40)
    at = pos[:, None].cpu() + torch.arange(300)
    cos, sin = _angles(at)
    q = plq.ops.rope_kv_append_fp8(qkv, cos, sin, 16, kv_heads, cache, pos)
    k, v = _rope(qkv.view(b, 300, -1, 128)[:, :, 16:24], cos[:, :, None], sin[:, :, None]), qkv.view(b, 300, -1, 128)[:, :, 24:]
    for i in (0, 2, 4):
        p = int(pos[i])
        for codes, scale, new in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v)):
            s = scale[i].repeat_interleave(BLOCK, -1)[:, p:p + 300].t()[..., None]
            got = codes[i, p:p + 300].view(torch.float8_e4m3fn).float() * s
            assert torch.all((got - new[i].float()).abs() <= torch.maximum(new[i].float().abs() * 2.0 ** -4, s * 2.0 ** -10))
    only = plq.kv_cache.Fp8Cache(*(x[4:] for x in (cache.k, cache.k_scale, cache.v, cache.v_scale)))
    out = plq.ops.fp8_cache_attention(q[:, -1:].contiguous(), cache, pos + 299 * (pos >= 0))
    _check_attention(out[4:], q[4:, -1:].contiguous(), only, [room - 1])
    plq.check_device_status()
