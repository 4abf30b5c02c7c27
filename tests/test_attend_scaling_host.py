"""Which scalings the attention forms take: with log2(e) they have to stay numbers (they become the scores' factor)."""
import ctypes

import pytest

from fastkv_amd._lib import FASTKV_EINVAL, FASTKV_EWORKSPACE, load

P = 1 << 20                                                       # an address that is only checked, never read
S2, S3 = ctypes.c_int64 * 2, ctypes.c_int64 * 3
Q, C = S3(4096, 128, 1024), S3(25600, 12800, 128)


@pytest.mark.parametrize("scaling,want", [(1e-45, FASTKV_EWORKSPACE), (0.1, FASTKV_EWORKSPACE), (2.3e38, FASTKV_EWORKSPACE), (2.4e38, FASTKV_EINVAL),
                                          (3e38, FASTKV_EINVAL), (float("inf"), FASTKV_EINVAL), (0.0, FASTKV_EINVAL), (float("nan"), FASTKV_EINVAL)])
def test_scaling(scaling, want):
    """2^128 / log2(e) = 2.36e38.  (The calls have no workspace: the next check is that one.)"""
    assert load().fastkv_window_attention(0, 2, 8, 2, 128, 4, P, Q, P, C, P, C, 100, P, 1, 1, 9, 2, scaling, P, P, 0, None) == want
    assert load().fastkv_shared_prefix_attention(0, 2, 8, 2, 128, 4, P, Q, P, S2(12800, 128), P, S2(12800, 128), 100, P, C, P, C, 100, P, 1, 1, scaling,
                                                 P, P, 0, None) == want
