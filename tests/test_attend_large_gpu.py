"""The attention forms at row counts whose B * H * T passes 2^24."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F16 = torch.float16


def test_a_batch_of_long_prompts():
    """4 x 131072 tokens of 32 heads: each request's rows are those of a call with that request alone."""
    from fastkv_amd import ops
    B, H, Hkv, D, T = 4, 32, 8, 64, 131072
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(B, h, T, D, generator=g, device="cuda", dtype=F16) for h in (H, Hkv, Hkv))
    got = ops.window_attention(q, k, v, window=100, sinks=2)
    for b in (0, 3):
        assert torch.equal(got[b:b + 1], ops.window_attention(q[b:b + 1], k[b:b + 1], v[b:b + 1], window=100, sinks=2))
    # its last tokens, as a chunk over the rest (cut otherwise: fp16 results within their rounding)
    tail = ops.window_attention(q[3:, :, -50:], k[3:], v[3:], window=100, sinks=2)
    # two results of the same formula, each within (2^-11 for p and 2^-11 for the rounding) of sum p |v| <= max |v|
    assert float((tail.float() - got[3:, -50:].float()).abs().max()) <= 4 * 2.0 ** -11 * float(v[3].float().abs().max())


def test_one_head_of_more_than_2_to_24_rows():
    """More queries than rows: the first ones see nothing, the last 100 see what they see in a call of their own."""
    from fastkv_amd import ops
    D, T, rows = 64, 2 ** 24 + 3, 100
    g = torch.Generator(device="cuda").manual_seed(2)
    one, k, v = (torch.randn(1, 1, r, D, generator=g, device="cuda", dtype=F16) for r in (1, rows, rows))
    got = ops.window_attention(one.expand(1, 1, T, D), k, v, window=30, sinks=2)
    want = ops.window_attention(one.expand(1, 1, rows, D), k, v, window=30, sinks=2)
    assert not bool(got[:, :-rows].any())
    assert float((got[:, -rows:].float() - want.float()).abs().max()) <= 4 * 2.0 ** -11 * float(v.float().abs().max())
    assert bool(got[:, -rows:].any(-1).all())
