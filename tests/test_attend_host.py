"""Refusals of the attention forms over a cache and of the penalties: the library's own checks (they come before any launch, so they run without
a GPU) and the front-ends'."""
import ctypes

import pytest
import torch

from fastkv_amd import ops
from fastkv_amd._lib import FASTKV_EINVAL, FASTKV_EUNSUPPORTED, FASTKV_EWORKSPACE, load

P = 1 << 20                                                       # an address that is only checked, never read
S3, S2 = ctypes.c_int64 * 3, ctypes.c_int64 * 2


def window(dtype=0, B=2, H=8, Hkv=2, D=128, T=4, q=P, qs=(4096, 128, 1024), k=P, ks=(2560000, 1280000, 128), v=P, vs=(2560000, 1280000, 128), rows=10000,
           length=P, step=1, advance=0, win=0, sinks=2, scaling=0.1, out=P, ws=P, nbytes=1 << 40):
    return load().fastkv_window_attention(dtype, B, H, Hkv, D, T, q, S3(*qs) if qs else None, k, S3(*ks), v, S3(*vs), rows, length, step, advance,
                                          win, sinks, scaling, out, ws, nbytes, None)


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(dtype=-1), dict(B=0), dict(H=7), dict(Hkv=0), dict(H=1), dict(T=0), dict(rows=0), dict(q=None),
                                 dict(k=P + 8), dict(v=0), dict(qs=None), dict(qs=(4096, 128, 1020)), dict(ks=(2560000, 1280001, 128)),
                                 dict(vs=(1, 8, 8)), dict(step=2), dict(step=-1), dict(advance=1, length=None), dict(win=-1), dict(sinks=-1),
                                 dict(scaling=0.0), dict(scaling=-1.0), dict(scaling=float("nan")), dict(scaling=float("inf")), dict(out=None),
                                 dict(out=P + 2), dict(ws=None), dict(ws=P + 4), dict(T=2 ** 30, H=64, Hkv=8)])
def test_window_attention_refuses(bad):
    assert window(**bad) == FASTKV_EINVAL


@pytest.mark.parametrize("D", [0, 32, 96, 192, 512])
def test_window_attention_head_dims(D):
    assert window(D=D) == (FASTKV_EINVAL if D == 0 else FASTKV_EUNSUPPORTED)


def test_window_attention_refuses_a_small_workspace():
    need = load().fastkv_attend_workspace_bytes(2, 8, 2, 128, 4, 10000, 0, 2, 0, 1)
    assert need > 0 and window(advance=1, nbytes=need - 1) == FASTKV_EWORKSPACE
    assert load().fastkv_attend_workspace_bytes(2, 8, 3, 128, 4, 100, 10, 2, 0, 1) == 0


def prefix(dtype=0, B=2, H=8, Hkv=2, D=128, T=4, kp=P, kps=(12800, 128), n=100, rows=100, length=P, scaling=0.1, nbytes=1 << 40, ws=P):
    s = S3(25600, 12800, 128)
    return load().fastkv_shared_prefix_attention(dtype, B, H, Hkv, D, T, P, S3(4096, 128, 1024), kp, S2(*kps), P, S2(12800, 128), n, P, s, P, s, rows,
                                                 length, 1, 0, scaling, P, ws, nbytes, None)


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(B=0), dict(H=9), dict(T=0), dict(kp=None), dict(kp=P + 8), dict(kps=(12800, 129)), dict(n=0),
                                 dict(n=-4), dict(rows=0), dict(length=None), dict(scaling=0.0), dict(ws=None)])
def test_shared_prefix_attention_refuses(bad):
    assert prefix(**bad) == FASTKV_EINVAL


def test_shared_prefix_attention_workspace():
    need = load().fastkv_attend_workspace_bytes(2, 8, 2, 128, 4, 100, 0, 0, 100, 0)
    assert need > 0 and prefix(nbytes=need - 1) == FASTKV_EWORKSPACE
    assert prefix(D=80) == FASTKV_EUNSUPPORTED


def penalties(dtype=0, B=2, V=100, x=P, row=100, tokens=P, trow=50, L=50, step=1, bias=None, brow=0, arow=0, out=2 * P, orow=100):
    return load().fastkv_decode_penalties(dtype, B, V, x, row, tokens, trow, L, P, step, P, 1, P, 1, P, 1, P, 1, bias, brow, None, arow, out, orow, None)


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(dtype=-1), dict(B=0), dict(B=70000), dict(V=0), dict(x=None), dict(row=99), dict(tokens=None),
                                 dict(tokens=P + 4), dict(trow=-1), dict(L=-1), dict(step=2), dict(brow=-8), dict(arow=-1), dict(out=None),
                                 dict(orow=50), dict(x=P + 1), dict(dtype=2, x=P + 2), dict(out=P + 2), dict(out=P, orow=104), dict(out=P + 200)])
def test_penalties_refuse(bad):
    assert penalties(**bad) == FASTKV_EINVAL


def test_front_ends_refuse_cpu_tensors():
    q, k = torch.zeros(1, 4, 1, 64, dtype=torch.float16), torch.zeros(1, 2, 9, 64, dtype=torch.float16)
    n = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.window_attention(q, k, k), lambda: ops.decode_window_attention(q, k, k, n, 0.1),
                 lambda: ops.decode_shared_prefix_attention(q, k, k, k, k, n, 0.1), lambda: ops.decode_penalties(torch.zeros(1, 8))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_penalties_front_end_checks_shapes():
    with pytest.raises(ValueError, match="logits"):
        ops.decode_penalties(torch.zeros(1, 2, 8))
    with pytest.raises(ValueError, match="logits"):
        ops.decode_penalties(torch.zeros(1, 8, dtype=torch.float64))
    with pytest.raises(ValueError, match="one token"):
        ops.decode_window_attention(torch.zeros(1, 4, 2, 64), torch.zeros(1, 2, 9, 64), torch.zeros(1, 2, 9, 64), None, 0.1)
