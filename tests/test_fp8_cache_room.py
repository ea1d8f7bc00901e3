"""How many positions an E4M3 cache holds, and what the decoder does behind them (host logic, on CPU tensors)."""
import types

import pytest
import torch

from plaquant_b200 import forward_pass, kv_cache


@pytest.fixture
def model():
    m = object.__new__(forward_pass.ResQForwardB200)
    m.kv_quant, m.kv_heads, m.device, m.layers, m.kv = "fp8", 2, torch.device("cpu"), [types.SimpleNamespace()], [None]
    return m


def _step(m, t, pos0, b=2):
    cache = m._fp8_room(0, b, t, pos0)
    assert cache.room >= pos0 + t and m.kv[0] is cache
    cache.appended(pos0, t)
    return cache


def test_positions_that_nobody_wrote_are_refused(model):
    """A prompt of 10 has room for more, but what lies there is anything."""
    cache = _step(model, 10, 0)
    assert cache.length == 10 and cache.room > 12
    for pos0 in (11, 12, cache.room - 1, cache.room, cache.room + 5, -1, -200):
        with pytest.raises(RuntimeError):
            model._fp8_room(0, 2, 1, pos0)
    assert model.kv[0] is cache and cache.length == 10
    assert _step(model, 1, 10).length == 11
    with pytest.raises(RuntimeError):
        model._fp8_room(0, 2, 1, 12)
    assert _step(model, 3, 5).length == 11                # back behind earlier positions: those after them stay written
    assert _step(model, 500, 11).length == 511            # a longer cache keeps what it held
    with pytest.raises(RuntimeError):
        model._fp8_room(0, 2, 1, 512)
    assert _step(model, 4, 0).length == 4                 # another prompt
    with pytest.raises(RuntimeError):
        model._fp8_room(0, 2, 1, 5)


def test_a_step_that_fails_before_its_append_adds_nothing(model):
    _step(model, 10, 0)
    model._fp8_room(0, 2, 4, 10)
    with pytest.raises(RuntimeError):
        model._fp8_room(0, 2, 1, 14)


def test_a_cache_put_back_keeps_its_length(model):
    kept = _step(model, 70, 0).clone()
    _step(model, 30, 70)
    assert kept.length == 70
    model.kv[0] = kept
    with pytest.raises(RuntimeError):
        model._fp8_room(0, 2, 1, 71)
    assert _step(model, 1, 70).length == 71
    grown = kept.grown(1000)
    assert grown.length == 71 and grown.room == 1000
    other = kv_cache.Fp8Cache.empty(2, 200, 2, "cpu", length=0)
    assert other.length == 0
    other.copy_from(kept, 33)
    assert other.length == 33
    other.copy_from(kept, 128)
    assert other.length == 71


def test_a_cache_of_the_callers_own_is_the_callers_to_answer_for(model):
    """Filled at positions in device memory, by copies or made from tensors: the host does not count, the room is the limit."""
    own = kv_cache.Fp8Cache.empty(2, 100, 2, "cpu")
    own.appended(0, 10)
    assert own.length is None
    cache = kv_cache.Fp8Cache.empty(2, 100, 2, "cpu", length=0)
    cache.appended(torch.tensor([5, 9]), 1)
    assert cache.length is None
    cache.appended(3, 1)
    assert cache.length is None
    made = kv_cache.Fp8Cache(cache.k, cache.k_scale, cache.v, cache.v_scale)
    assert made.length is None and made.clone().length is None
    for c in (own, cache, made):
        model.kv[0] = c
        assert model._fp8_room(0, 2, 1, 99) is c
        with pytest.raises(RuntimeError):
            model._fp8_room(0, 2, 1, 101)
    old = object.__new__(kv_cache.Fp8Cache)               # pickled before there was a length
    old.__dict__.update(k=cache.k, k_scale=cache.k_scale, v=cache.v, v_scale=cache.v_scale)
    assert old.length is None and old.clone().length is None


def test_an_append_with_a_gap_leaves_the_length():
    cache = kv_cache.Fp8Cache.empty(1, 100, 1, "cpu", length=0)
    cache.appended(4, 10)
    assert cache.length == 0
    cache.appended(-1, 10)
    assert cache.length == 0
    cache.appended(0, 4)
    cache.appended(4, 10)
    assert cache.length == 14


@pytest.mark.parametrize("value", [False, True, None, 0, 1, 2, "", "fp8", "fake", "nvfp4"])
def test_forms_of_the_cache_that_were_accepted_before(value):
    forward_pass.ResQForwardB200._check_kv_quant(value)


@pytest.mark.parametrize("value", ["fp9", "fp4", "fp8_e5m2"])
def test_forms_of_the_cache_that_do_not_exist(value):
    with pytest.raises(ValueError):
        forward_pass.ResQForwardB200._check_kv_quant(value)


def test_a_cache_without_heads_is_refused():
    with pytest.raises(TypeError):
        kv_cache.Fp8Cache.empty(1, 64, 0, "cpu").check(1, 0, torch.device("cpu"))
