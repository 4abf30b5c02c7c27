"""FASTKV_WINDOW_ATTENTION=1 where a prompt's mask holds more than the window: SDPA's answer stays."""
import pytest
import torch

from test_window_decode_gpu import IDS, build

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("given", ["hole", "ones", "none", "positions"])
def test_a_mask_that_hides_tokens_stays_with_sdpa(monkeypatch, given):
    """A window of 100 over 600 tokens; "hole": the mask hides tokens 530 .. 569, which the last tokens' window holds.  Behind the token selection
    (layer 0) the reference masks the kept tokens by the window alone, so layer 1 may take the kernel."""
    from fastkv_amd import ops
    model, _ = build(monkeypatch, "0", 100)
    ids = IDS.cuda()
    kw = dict(attention_mask=torch.ones_like(ids))
    if given == "hole":
        kw["attention_mask"][:, 530:570] = 0
    elif given == "none":
        kw = {}
    elif given == "positions":                                    # two sequences side by side, no cache: the mask builder keeps them apart
        kw = dict(position_ids=torch.cat([torch.arange(560), torch.arange(40)])[None].cuda(), use_cache=False)
    calls = []
    real = ops.window_attention
    monkeypatch.setattr(ops, "window_attention", lambda *a, **k: calls.append(a[0].shape[2]) or real(*a, **k))
    with torch.no_grad():
        want = model(ids, **kw).logits.float()
        assert not calls
        monkeypatch.setenv("FASTKV_WINDOW_ATTENTION", "1")
        got = model(ids, **kw).logits.float()
    if given == "positions":
        assert not calls and torch.equal(got, want)               # no cache: no token selection either, two layers of SDPA
        return
    assert calls == ([256] if given == "hole" else [600, 256])
    assert float((got - want).abs().max()) <= 2e-2 * float(want.abs().max())          # as the decode paths are compared
