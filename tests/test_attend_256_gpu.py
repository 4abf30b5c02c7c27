"""Head size 256, whose kernels are cut by rules of their own: the requests' rows packed beside single tokens, several packed tokens per request,
and the join of eight slices and more (tests/attend_ref.py derives the tolerance)."""
import pytest
import torch

from attend_ref import attend, check, prefix_rows, window_rows
from test_attend_gpu import dev_lens, make

pytestmark = pytest.mark.gpu
F16, BF16, D = torch.float16, torch.bfloat16, 256


def slots(B, H, Hkv, T, rows, window, sinks, P, advance):
    """Slices per row that the call's workspace has room for ({m, l} and 256 sums each)."""
    from fastkv_amd._lib import load
    need = load().fastkv_attend_workspace_bytes(B, H, Hkv, D, T, rows, window, sinks, P, advance)
    assert need % (B * H * T * (D + 2) * 4) == 0
    return need // (B * H * T * (D + 2) * 4)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,H,Hkv,T,P,rows,lens,least", [
    (16, 32, 8, 1, 2048, 40, [i * 2 for i in range(16)], 8),       # 64 packed rows beside single tokens, many slices
    (35, 8, 2, 1, 333, 12, [i % 12 for i in range(35)], 2),        # 140 packed rows: a ragged last tile
    (34, 4, 4, 1, 70, 9, [-1 if i == 5 else i % 9 for i in range(34)], 2),   # one row per request, one idle
    (3, 8, 2, 5, 200, 60, [0, 17, 55], 2),                         # several tokens: 60 packed rows
    (5, 8, 2, 9, 1500, 64, [-4, 55, 20, 1, 0], 8),                 # 180 packed rows, left padding, many slices
    (2, 6, 2, 17, 90, 1700, [1600, 30], 2),                        # own rows far longer than the prefix
    (2, 8, 2, 33, 300, 50, [3, 17], 0),                            # 132 rows per request: no packing
])
def test_shared_prefix(B, H, Hkv, T, P, rows, lens, least, dtype):
    from fastkv_amd import ops
    assert slots(B, H, Hkv, T, rows, 0, 0, P, 0) >= least
    q, k, v = make(B + T, B, H, Hkv, D, T, rows, dtype)
    _, kp, vp = make(B + T + 1, 1, H, Hkv, D, 1, P, dtype)
    for b in range(B):                                             # nobody reads rows behind a request's own end
        k[b, :, max(0, lens[b] + T):] = float("nan")
        v[b, :, max(0, lens[b] + T):] = float("nan")
    n = dev_lens(lens)
    args = (q.cuda(), kp.cuda(), vp.cuda(), k.cuda(), v.cuda(), n, D ** -0.5)
    ref, bound = attend(q, prefix_rows(kp[0].double(), vp[0].double(), k.double(), v.double(), lens, T, Hkv, H), D ** -0.5)
    check(ops.decode_shared_prefix_attention(*args, advance=False), ref, bound)
    check(ops.decode_shared_prefix_attention(*args), ref, bound)
    assert n.tolist() == [x + T if x >= 0 else x for x in lens]


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_infinities_that_some_of_several_packed_tokens_see(dtype):
    from fastkv_amd import ops
    B, H, Hkv, T, P, rows, lens = 4, 8, 2, 6, 130, 80, [70, 0, 33, 8]
    q, k, v = make(9, B, H, Hkv, D, T, rows, dtype)
    _, kp, vp = make(10, 1, H, Hkv, D, 1, P, dtype)
    v[0, 0, 72, 200] = float("nan")                                # tokens 2 .. 5 of request 0
    v[2, 1, 38] = float("inf")                                     # the last token of request 2
    k[3, 0, 10, 0] = float("nan")                                  # tokens 2 .. 5 of request 3
    vp[0, 1, 129, 7] = -float("inf")                               # everybody, in the prefix' last, partly filled tile
    got = ops.decode_shared_prefix_attention(q.cuda(), kp.cuda(), vp.cuda(), k.cuda(), v.cuda(), dev_lens(lens), D ** -0.5, advance=False)
    ref, bound = attend(q, prefix_rows(kp[0].double(), vp[0].double(), k.double(), v.double(), lens, T, Hkv, H), D ** -0.5)
    assert torch.isfinite(ref).any() and not torch.isfinite(ref).all()
    check(got, ref, bound)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,H,Hkv,T,rows,window,sinks,lens,least", [
    (1, 32, 8, 1, 2500, 2048, 4, [2400], 8),                       # one request's token: the join of many slices
    (2, 12, 4, 1, 3000, 1111, 100, [2999, 50], 2),
    (1, 6, 2, 2, 2300, 2047, 0, [2290], 8),                        # two tokens
    (2, 4, 1, 150, 900, 600, 5, [700, 0], 0),                      # a chunk
])
def test_window(B, H, Hkv, T, rows, window, sinks, lens, least, dtype):
    from fastkv_amd import ops
    assert slots(B, H, Hkv, T, rows, window, sinks, 0, 0) >= least
    q, k, v = make(T, B, H, Hkv, D, T, rows, dtype)
    for b in range(B):
        k[b, :, lens[b] + T:] = float("nan")
        v[b, :, lens[b] + T:] = float("nan")
    got = ops.window_attention(q.cuda(), k.cuda(), v.cuda(), window=window, sinks=sinks, len_dev=dev_lens(lens))
    ref, bound = attend(q, window_rows(k.double(), v.double(), lens, T, window, sinks, Hkv, H), D ** -0.5)
    check(got, ref, bound)
    if T == 1:
        n = dev_lens(lens)
        check(ops.decode_window_attention(q.cuda(), k.cuda(), v.cuda(), n, D ** -0.5, window=window, sinks=sinks), ref, bound)
        assert n.tolist() == [min(x + 1, rows) for x in lens]
