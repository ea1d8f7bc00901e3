"""The decoder on the E4M3 cache and head: positions it does not hold, and what the options leave on the device."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def plq():
    import plaquant_b200
    return plaquant_b200


def _config(**kw):
    from plaquant_b200.forward_pass import LlamaConfig
    return LlamaConfig(**{**dict(hidden_size=512, intermediate_size=1024, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=128, vocab_size=1003), **kw})


def _ids(cfg, b, t, seed=1):
    return torch.randint(0, cfg.vocab_size, (b, t), generator=torch.Generator().manual_seed(seed)).cuda()


def test_a_gap_behind_the_prompt_is_refused(plq):
    from plaquant_b200.forward_pass import ResQForwardB200
    cfg = _config()
    m = ResQForwardB200(cfg, "cuda", seed=6, kv_quant="fp8")
    ids = _ids(cfg, 2, 40)
    m.forward(ids[:, :20])
    assert [c.length for c in m.kv] == [20, 20] and m.kv[0].room > 30
    for pos0 in (21, 30, -1):
        with pytest.raises(RuntimeError):
            m.forward(ids[:, 20:21], pos0=pos0)
    kept = [c.clone() for c in m.kv]
    a = m.forward(ids[:, 20:30], pos0=20)
    assert m.kv[0].length == 30
    m.kv = kept
    assert torch.equal(m.forward(ids[:, 20:30], pos0=20), a)
    again = m.forward(ids[:, 20:30], pos0=20)             # the same positions once more
    assert again.isfinite().all() and m.kv[1].length == 30
    plq.check_device_status()


def test_the_append_keeps_the_length(plq):
    from plaquant_b200 import kv_cache
    cache = kv_cache.Fp8Cache.empty(1, 100, 1, "cuda", length=0)
    qkv, one = torch.ones(1, 5, 3 * 128, dtype=torch.bfloat16, device="cuda"), torch.ones(5, 128, device="cuda")
    plq.ops.rope_kv_append_fp8(qkv, one, one, 1, 1, cache, 0)
    plq.ops.rope_kv_append_fp8(qkv, one, one, 1, 1, cache, 5)
    assert cache.length == 10
    with pytest.raises(plq.PlqError):
        plq.ops.rope_kv_append_fp8(qkv, one, one, 1, 1, cache, 96)
    assert cache.length == 10
    plq.ops.rope_kv_append_fp8(qkv, one, one, 1, 1, cache, torch.tensor([10], device="cuda"))
    assert cache.length is None


@pytest.mark.parametrize("value,same_as", [(None, False), (0, False), (1, True), ("nvfp4", True)])
def test_other_words_for_the_older_caches(plq, monkeypatch, value, same_as):
    """None and other false values are the bf16 cache, other true ones the packed rows, on the same native call."""
    from plaquant_b200 import _lib
    from plaquant_b200.forward_pass import ResQForwardB200
    cfg, calls = _config(), []
    front = _lib.torch_lib()
    layer = front.decoder_layer
    monkeypatch.setattr(front, "decoder_layer", lambda *a: (calls.append(1), layer(*a))[1])
    ids, got = _ids(cfg, 2, 30), []
    for v in (value, same_as):
        m = ResQForwardB200(cfg, "cuda", seed=6, kv_quant=v)
        got.append((m.forward(ids[:, :29]), m.forward(ids[:, 29:], pos0=29), m.generate(ids, 5), m.kv_quant))
        assert len(calls) % 2 == 0 and calls
    assert all(torch.equal(x, y) for x, y in zip(got[0][:3], got[1][:3])) and got[0][3] is value


def test_the_quantised_head_takes_the_place_of_the_other(plq, tmp_path):
    """Half of the bytes stay on the device; the container written from such a model holds the head as it was."""
    from plaquant_b200 import weight_packer
    from plaquant_b200.forward_pass import ResQForwardB200
    cfg = _config(vocab_size=40000)
    ids, sizes, models = _ids(cfg, 2, 20), [], []
    for fp8_head in (False, True):
        before = torch.cuda.memory_allocated()
        models.append(ResQForwardB200(cfg, "cuda", seed=6, fp8_head=fp8_head))
        sizes.append(torch.cuda.memory_allocated() - before)
    plain, m = models
    head = 40000 * 512
    assert sizes[0] - sizes[1] >= head - head // 1024 - 4096 and m.lm_head.device.type == "cpu"
    assert torch.equal(m.lm_head, plain.lm_head.cpu())
    state = weight_packer.read_packed(weight_packer.save_packed(m, str(tmp_path / "m.pt")))
    again = ResQForwardB200(cfg, "cuda", packed=state, fp8_head=True)
    assert torch.equal(again.forward(ids), m.forward(ids)) and again.lm_head.device.type == "cpu"
    assert torch.equal(ResQForwardB200(cfg, "cuda", packed=state).forward(ids), plain.forward(ids))


def test_no_queries_in_front_of_nothing(plq):
    """T = 0 at position 0, as at any other, and no sequences."""
    from plaquant_b200 import kv_cache
    for b in (0, 2):
        cache = kv_cache.Fp8Cache.empty(b, 64, 2, "cuda")
        for pos in (0, 3, torch.zeros(b, dtype=torch.int64, device="cuda")):
            q = torch.empty(b, 0, 8, 128, dtype=torch.bfloat16, device="cuda")
            assert plq.ops.fp8_cache_attention(q, cache, pos).shape == (b, 0, 8, 128)
            none = torch.empty(0, 128, device="cuda")
            assert plq.ops.rope_kv_append_fp8(torch.empty(b, 0, 12 * 128, dtype=torch.bfloat16, device="cuda"), none, none, 8, 2, cache, pos).shape == q.shape
    plq.check_device_status()


@pytest.mark.parametrize("heads,kv_heads,fp8_head", [(4, 2, False), (4, 4, True), (18, 2, False)])
def test_layer_calls_around_the_cache_equal_the_operator_path(plq, monkeypatch, heads, kv_heads, fp8_head):
    """Prompts of up to 16 rows and more, a chunk, single steps, a captured decode; the caches as well."""
    from plaquant_b200 import _lib, forward_pass
    cfg = _config(hidden_size=heads * 128, num_heads=heads, num_kv_heads=kv_heads)
    ids = _ids(cfg, 3, 40, seed=7)
    m = forward_pass.ResQForwardB200(cfg, "cuda", seed=3, kv_quant="fp8", fp8_head=fp8_head)
    front, calls = _lib.torch_lib(), []
    back = front.layer_back
    monkeypatch.setattr(front, "layer_back", lambda *a: (calls.append(1), back(*a))[1])

    def everything():
        out = [m.forward(ids[:, :21]), m.forward(ids[:, 21:24], pos0=21)]
        out += [m.forward(ids[:, i:i + 1], pos0=i) for i in range(24, 28)]
        out += [x for c in m.kv for x in (c.k[:, :28].clone(), c.k_scale[..., 0].clone(), c.v[:, :28].clone(), c.v_scale[..., 0].clone())]
        m._decode_states.clear()
        return out + [m.generate(ids[:, :9], 5), m.forward(ids[:, :9], all_positions=True), m.forward(ids[:, :1]), m.forward(ids[:1, :5])]
    got = everything()
    n = len(calls)
    assert n >= 2 * 12
    monkeypatch.setattr(forward_pass, "NATIVE_LAYER_ROWS", 0)
    want = everything()
    assert len(calls) == n and all(torch.equal(a, b) for a, b in zip(got, want)) and len(got) == len(want)
    with pytest.raises(RuntimeError):
        back(m.layers[0].o.native(), m.layers[0].gate_up.native(), m.layers[0].down.native(), m.layers[0].ln2, 1e-6,
             torch.zeros(1, 2, heads * 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 3, heads * 128, dtype=torch.bfloat16, device="cuda"), False)
    with pytest.raises(RuntimeError):
        front.layer_front(m.layers[0].qkv.native(), m.layers[0].ln1, 1e-6, torch.zeros(1, 2, 128, dtype=torch.bfloat16, device="cuda"), None)
    plq.check_device_status()
