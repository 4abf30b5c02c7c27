"""Where the penalties' result may not go: the library's own checks, which come before any launch."""
import pytest

from fastkv_amd._lib import FASTKV_EINVAL, load

P = 1 << 20                                                       # addresses that are only checked, never read
B, V, L = 3, 100, 50


def penalties(out, orow=V, x=P, row=V, tokens=8 * P, n=9 * P, rep=10 * P, freq=11 * P, bias=12 * P, brow=V, allowed=13 * P, arow=4, dtype=2):
    return load().fastkv_decode_penalties(dtype, B, V, x, row, tokens, L, L, n, 1, None, 0, rep, 1, None, 0, freq, 0, bias, brow, allowed, arow, out, orow,
                                          None)


@pytest.mark.parametrize("bad", [
    dict(out=12 * P), dict(out=12 * P, brow=0), dict(out=12 * P, x=12 * P), dict(out=12 * P + 4 * (V - 1)),       # the bias, and its last element
    dict(out=13 * P), dict(out=8 * P + 8), dict(out=9 * P), dict(out=10 * P + 8), dict(out=11 * P - 4 * (3 * V - 1)),
    dict(out=P + 4 * V, orow=2 * V, row=2 * V - 1),               # rows that meet, of other strides
    dict(out=P + 4 * (V - 1), orow=2 * V, row=2 * V),             # one element of the next row
    dict(out=P - 4 * (V - 1), orow=2 * V, row=2 * V),
    dict(out=P + 4 * (2 * V - 1), orow=2 * V, row=2 * V),
])
def test_out_may_not_be_what_is_read(bad):
    assert penalties(**bad) == FASTKV_EINVAL
