"""Refusals of the append in front of the attention forms over a cache: the library's own checks (they come before any launch, so they
run without a GPU) and the front-end's."""
import ctypes

import pytest
import torch

from fastkv_amd import ops
from fastkv_amd._lib import FASTKV_EINVAL, FASTKV_EUNSUPPORTED, load

P = 1 << 20                                                       # an address that is only checked, never read
S2, S3 = ctypes.c_int64 * 2, ctypes.c_int64 * 3


def append(B=2, Hkv=2, D=128, k=P, ks=(256, 128), v=P, vs=(256, 128), kslab=P, vslab=P, ss=(12800, 6400, 128), rows=50, length=P, step=1):
    return load().fastkv_decode_append(B, Hkv, D, k, S2(*ks), v, S2(*vs), kslab, vslab, S3(*ss), rows, length, step, None)


@pytest.mark.parametrize("bad", [dict(step=2), dict(step=-1), dict(length=None), dict(B=0), dict(Hkv=0), dict(rows=0), dict(k=None), dict(v=P + 8),
                                 dict(kslab=None), dict(vslab=P + 2), dict(ks=(250, 128)), dict(vs=(256, 4)), dict(ss=(12800, 6400, 100))])
def test_append_refuses(bad):
    assert append(**bad) == FASTKV_EINVAL


def test_append_head_dims():
    assert append(D=80) == FASTKV_EUNSUPPORTED


def test_front_end_refuses_other_types_and_lengths():
    slab, new = torch.zeros(3, 2, 9, 64, dtype=torch.float16), torch.zeros(3, 2, 1, 64, dtype=torch.float16)
    n = torch.zeros(3, dtype=torch.int32)
    for a in ((slab, slab, new.bfloat16(), new), (slab, slab.bfloat16(), new, new), (slab.float(),) * 2 + (new.float(),) * 2):
        with pytest.raises(TypeError, match="one type, fp16 or bf16"):
            ops.decode_append(*a, n)
    for bad in (n.long(), n[:2], torch.zeros(6, dtype=torch.int32)[::2], n[:, None]):
        with pytest.raises(ValueError, match="1 or 3 lengths"):
            ops.decode_append(slab, slab, new, new, bad)
    for good in (n, n[:1], n[0]):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            ops.decode_append(slab, slab, new, new, good)


def test_the_dense_decode_refuses_a_length_per_request():
    """It reads and advances the first length alone."""
    q, new, slab = (torch.zeros(3, h, r, 64, dtype=torch.float16) for h, r in ((4, 1), (2, 1), (2, 9)))
    n, cos = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 1, 64, dtype=torch.float16)
    for bad in (n, n[:1].long()):
        with pytest.raises(ValueError, match="one int32 length"):
            ops.decode_attention(q, slab, slab, bad, 0.1)
        with pytest.raises(ValueError, match="one int32 length"):
            ops.decode_step_attention(q, new, new, cos, cos, slab, slab, bad, 0.1)
