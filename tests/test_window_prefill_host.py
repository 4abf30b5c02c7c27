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
