"""The E4M3 operators where the package uses them: the linear, the LM head and the cache of the decoder, together."""
import pytest
import torch

from tests._util import synth_activation, synth_gamma, synth_weight

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def plq():
    import plaquant_b200
    return plaquant_b200


def _config(**kw):
    from plaquant_b200.forward_pass import LlamaConfig
    return LlamaConfig(**{**dict(hidden_size=512, intermediate_size=1024, num_layers=3, num_heads=4, num_kv_heads=2, head_dim=128, vocab_size=1003), **kw})


def _cosine(a, b):
    return float(torch.nn.functional.cosine_similarity(a.double().flatten(), b.double().flatten(), dim=0))


@pytest.mark.parametrize("rows", [1, 40, 300])
@pytest.mark.parametrize("norm", [False, True])
def test_linear(plq, rows, norm):
    from plaquant_b200.quantize import Fp8Linear
    k, n = 1040, 384
    x, w = synth_activation(rows, k, seed=rows).cuda(), synth_weight(n, k, seed=9).cuda()
    gamma = synth_gamma(k, seed=3).cuda() if norm else None
    lin = Fp8Linear.from_weight(w)
    assert (lin.in_features, lin.out_features) == (k, n)
    y = lin(x.view(1, rows, k), norm_weight=gamma)
    assert y.shape == (1, rows, n) and torch.equal(y.view(rows, n), plq.fp8_gemm(plq.fp8_pack(x, gamma=gamma), plq.fp8_pack_weight(w)))
    assert torch.equal(lin(lin.quantize_input(x, gamma)), y.view(rows, n))
    out = torch.empty(rows, n, dtype=torch.float32, device="cuda")
    assert torch.equal(lin(x, norm_weight=gamma, out=out), lin(x, norm_weight=gamma, out_dtype=torch.float32))
    # both operands off by at most 2^-4 of themselves, signs at random: sqrt(2) * 2^-4 / sqrt(3) of the result on average
    f = x.double() if gamma is None else gamma.double() * x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + 1e-6)
    want = f @ w.double().t()
    assert float((out.double() - want).norm() / want.norm()) <= 2 ** 0.5 * 2.0 ** -4
    cpu = Fp8Linear(lin.weight.codes.cpu(), lin.weight.scales.cpu())
    with pytest.raises(RuntimeError):
        cpu(x)
    assert torch.equal(cpu.to("cuda")(x), lin(x))


@pytest.mark.parametrize("b,t", [(1, 1), (3, 5), (2, 40)])
def test_lm_head(plq, b, t):
    """fp8_head: the same stack, logits from the quantised norm and head, whether or not the last add is part of the quantiser."""
    from plaquant_b200.forward_pass import ResQForwardB200
    cfg = _config()
    plain, m = ResQForwardB200(cfg, "cuda", seed=5), ResQForwardB200(cfg, "cuda", seed=5, fp8_head=True)
    ids = torch.randint(0, cfg.vocab_size, (b, t), generator=torch.Generator().manual_seed(1)).cuda()
    every = m.forward(ids, all_positions=True)
    assert every.dtype == torch.float32 and every.shape == (b, t, cfg.vocab_size)
    h = torch.nn.functional.embedding(ids, m.embed)
    m.kv = [None] * len(m.layers)
    h, delta = m._run_layers(h, 0, m._rope_rows(0, t))
    p = plq.fp8_pack(h + delta, gamma=m.final_norm, eps=cfg.rms_eps)
    want = plq.fp8_gemm(p, m.head8.weight, out_dtype=torch.float32).view(b, t, -1)
    assert torch.equal(every, want) and torch.equal(m._logits(h + delta), want)
    ref = plain.forward(ids, all_positions=True)
    assert float((every - ref).norm() / ref.norm()) <= 2 ** 0.5 * 2.0 ** -4
    last = m.forward(ids)
    assert last.shape == (b, cfg.vocab_size) and _cosine(last, every[:, -1]) > 0.99


@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (4, 4), (4, 1)])
def test_decoder_with_the_cache(plq, monkeypatch, heads, kv_heads):
    """A prompt, single tokens and a chunk behind it: the cache holds the first layer's keys and values in 8 bits, and the
    attention is that of the positions in front of each query.  (What a layer's 4-bit linears make of it is not compared: they
    send any other rounding another way.)"""
    from plaquant_b200 import ops
    from plaquant_b200.forward_pass import ResQForwardB200
    cfg = _config(num_heads=heads, num_kv_heads=kv_heads, num_layers=1)
    m, ref = ResQForwardB200(cfg, "cuda", seed=6, kv_quant="fp8"), ResQForwardB200(cfg, "cuda", seed=6)
    ids = torch.randint(0, cfg.vocab_size, (2, 200), generator=torch.Generator().manual_seed(2)).cuda()
    seen = []
    attend = ops.fp8_cache_attention

    def watched(q, cache, pos, **kw):
        out = attend(q, cache, pos, **kw)
        seen.append((q.clone(), pos, out.clone()))
        return out
    monkeypatch.setattr(ops, "fp8_cache_attention", watched)
    at = 0
    for n in (70, 1, 1, 57, 1, 70):
        got, want = m.forward(ids[:, at:at + n], pos0=at), ref.forward(ids[:, at:at + n], pos0=at)
        assert got.shape == want.shape and got.isfinite().all()
        (q, pos, out), at = seen.pop(), at + n
        assert pos == at - n and not seen
        k, v = (x.double().repeat_interleave(heads // kv_heads, 2).transpose(1, 2) for x in m.kv[0].values(at))
        score = (q.double().transpose(1, 2) @ k.transpose(-1, -2)) * 128 ** -0.5
        score = score.masked_fill(torch.arange(at, device="cuda") > pos + torch.arange(n, device="cuda")[:, None], float("-inf"))
        exact = (torch.softmax(score, -1) @ v).transpose(1, 2)
        # weights of at least 8 bits (2^-8), the rounding of the result (2^-8), fixed steps and scores well below either
        assert torch.all((out.double() - exact).abs() <= 2.0 ** -8 * exact.abs() + (2.0 ** -8 + 2.0 ** -10) * v.abs().amax())
        for mine, theirs in zip(m.kv[0].values(at), ref.kv[0]):
            # the same projections in E4M3: off by 2^-4, or by half a step where the block's largest value is at 224 .. 448
            scale = theirs.float().abs().amax()
            assert torch.all((mine.float() - theirs.float()).abs() <= torch.maximum(theirs.float().abs() * 2.0 ** -4, scale * 2.0 ** -9 / 224) * (1 + 2.0 ** -6))
    kept = m.kv[0].clone()
    m.forward(ids[:, :1], pos0=at)
    assert torch.equal(kept.k[:, :at // 64 * 64], m.kv[0].k[:, :at // 64 * 64])
    m.kv[0] = None
    with pytest.raises(RuntimeError):
        m.forward(ids[:, :1], pos0=at)
    with pytest.raises(ValueError):
        ResQForwardB200(cfg, "cuda", kv_quant="fp9")
    plq.check_device_status()


def test_generation_in_a_graph_equals_the_steps_one_by_one(plq):
    from plaquant_b200.forward_pass import ResQForwardB200
    cfg = _config()
    m = ResQForwardB200(cfg, "cuda", seed=7, kv_quant="fp8", fp8_head=True)
    ids = torch.randint(0, cfg.vocab_size, (3, 33), generator=torch.Generator().manual_seed(3)).cuda()
    steps = m.generate(ids, 40, use_graph=False)
    for _ in range(2):                                  # captured, and replayed from the kept graph
        assert torch.equal(m.generate(ids, 40), steps)
    other = torch.randint(0, cfg.vocab_size, (1, 90), generator=torch.Generator().manual_seed(4)).cuda()
    assert torch.equal(m.generate(other, 7), m.generate(other, 7, use_graph=False))
    plq.check_device_status()


def test_objects_of_before_have_no_such_head():
    from plaquant_b200.forward_pass import ResQForwardB200
    old = ResQForwardB200.__new__(ResQForwardB200)
    assert old.head8 is None
