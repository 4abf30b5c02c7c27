"""Which prompts the windowed prefill attention takes (FASTKV_WINDOW_ATTENTION=1)."""
import types

import pytest
import torch

from baselines.fastkv import _wiring


@pytest.mark.parametrize("mask,packed,takes", [
    (None, False, True), (torch.ones(2, 9, dtype=torch.int64), False, True), (torch.ones(2, 9, dtype=torch.bool), False, True),
    (torch.tensor([[0, 1, 1], [1, 1, 1]]), False, False), (torch.tensor([[True, True, False]]), False, False),
    (torch.zeros(1, 1, 3, 3), False, False), ({"sliding_attention": torch.ones(1, 3)}, False, False), (None, True, False),
    (torch.ones(1, 3), True, False)])
def test_only_a_window_alone(monkeypatch, mask, packed, takes):
    config = types.SimpleNamespace(sliding_window=64)
    assert not _wiring._window_alone(config, mask, packed)        # not asked for
    monkeypatch.setenv("FASTKV_WINDOW_ATTENTION", "1")
    assert _wiring._window_alone(config, mask, packed) is takes
    assert not _wiring._window_alone(types.SimpleNamespace(sliding_window=None), mask, packed)
    assert not _wiring._window_alone(types.SimpleNamespace(), mask, packed)


@pytest.mark.parametrize("trained", ["q", "k", "v", None])
def test_a_gradient_of_any_projection_keeps_sdpa(trained):
    """An adapter on the key or value projection alone: the kernel has no backward pass, and refuses."""
    states = [types.SimpleNamespace(is_cuda=True, dtype=torch.float16, shape=(1, 4, 9, 64), requires_grad=n == trained) for n in "qkv"]
    assert _wiring._prefill_window(*states) is (trained is None)
    with torch.no_grad():
        assert _wiring._prefill_window(*states)


@pytest.mark.parametrize("dtype,D,fits", [(torch.float16, 64, True), (torch.bfloat16, 128, True), (torch.float16, 256, True), (torch.float32, 64, False),
                                          (torch.float16, 96, False)])
def test_static_decode_over_a_window_is_refused_up_front_where_its_kernel_does_not_take_the_slabs(dtype, D, fits):
    slab = lambda rows: types.SimpleNamespace(kslab=torch.empty(1, 2, rows, D, dtype=dtype))      # noqa: E731
    cache = types.SimpleNamespace(layers=[slab(300), types.SimpleNamespace(kslab=None), slab(200)])
    for config in (types.SimpleNamespace(sliding_window=None), types.SimpleNamespace(sliding_window=300), types.SimpleNamespace()):
        _wiring._require_window_decode(config, cache)             # no window that the slabs outgrow
    small = types.SimpleNamespace(sliding_window=256)
    if fits:
        _wiring._require_window_decode(small, cache)
    else:
        with pytest.raises(ValueError, match="sliding_window = 256"):
            _wiring._require_window_decode(small, cache)


def test_the_model_asks_before_its_first_layer():
    from transformers.models.mistral.modeling_mistral import MistralModel

    from baselines.monkeypatch import replace_mistral
    from fastkv_amd.cache import FastKVSlabCache
    replace_mistral("fastkv")
    config = types.SimpleNamespace(sliding_window=24, use_cache=True)
    cache = FastKVSlabCache(1)
    cache.layers[0].kslab = torch.zeros(1, 8, 40, 128)
    cache.layers[0].len, cache.layers[0].static_decode = 30, True
    model = types.SimpleNamespace(config=config, embed_tokens=lambda ids: torch.zeros(1, 1, 64), layers=None)
    with pytest.raises(ValueError, match="sliding_window = 24"):
        MistralModel.forward(model, input_ids=torch.zeros(1, 1, dtype=torch.int64), past_key_values=cache, position_ids=torch.full((1, 1), 30))
