"""Logits and result as parts of one wide tensor (tests/test_penalties_gpu.py has the formula and its tolerance)."""
import pytest
import torch

from test_penalties_gpu import call, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,gap", [(1000, 0), (999, 3)])
@pytest.mark.parametrize("swap", [False, True])
def test_rows_of_one_wide_tensor(V, gap, swap, dtype):
    """The logits in one half, the result in the other: no byte is in both, whichever comes first."""
    from fastkv_amd import ops
    s = make(V, 3, V, 60, dtype)
    want = call(ops, s)
    wide = torch.full((3, 2 * V + gap), float("nan"), dtype=dtype, device="cuda")
    left, right = wide[:, :V], wide[:, V + gap:]
    x, out = (right, left) if swap else (left, right)
    x.copy_(s["x"])
    d = {k: t.cuda() for k, t in s.items()}
    got = ops.decode_penalties(x, d["tokens"], d["n"], d["n0"], d["rep"], d["pres"], d["freq"], d["bias"], d["allowed"], out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out, want) and torch.equal(x.cpu(), s["x"])
    if gap:
        assert bool(torch.isnan(wide[:, V:V + gap]).all())
    from fastkv_amd._lib import FASTKV_EINVAL, FastKVNativeError
    with pytest.raises(FastKVNativeError) as e:                   # the bias is the result's memory: refused
        ops.decode_penalties(d["x"].float(), bias=d["bias"], out=d["bias"])
    assert e.value.code == FASTKV_EINVAL
