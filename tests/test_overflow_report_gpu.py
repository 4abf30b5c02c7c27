"""A full cache is reported, also where the first call of a process that could report it is recorded into a graph."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

# a process of its own: nothing of the library has run in it that reports anything
CHILD = """
import torch
from fastkv_amd import ops
from fastkv_amd._lib import FASTKV_EOVERFLOW, FastKVNativeError
D, rows = 64, 20
q, k, v = (torch.randn(1, h, r, D, device="cuda").half() for h, r in ((4, 1), (2, rows), (2, rows)))
n = torch.tensor([rows - 3], dtype=torch.int32, device="cuda")
slab = torch.randn(1, 2, 4096, D, device="cuda").half()
m = torch.full((1,), 4090, dtype=torch.int32, device="cuda")
ops.decode_window_attention(q, slab, slab, m, 0.125, advance=False)            # (loads the kernels; moves nothing on, reports nothing)
call = {call}
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    out = call()
torch.cuda.current_stream().wait_stream(side)
full = 0
for i in range(8):
    graph.replay()
    torch.cuda.synchronize()
    assert n.tolist() == [min(rows, rows - 2 + i)], (i, n)
    q.abs().sum()                                                             # the program's own work between the replays
    try:
        ops.raise_if_aborted()
        assert i < 3, i
    except FastKVNativeError as e:
        assert e.code == FASTKV_EOVERFLOW and i >= 3, i
        full += 1
assert full == 5
print("reported", full)
"""


@pytest.mark.parametrize("call", [
    "lambda: ops.decode_window_attention(q, k, v, n, 0.125, window=7, sinks=1)",
    "lambda: ops.decode_shared_prefix_attention(q, slab[0, :, :50], slab[0, :, :50], k, v, n, 0.125)",
])
def test_the_first_call_that_moves_a_length_may_be_captured(call):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CHILD.format(call=call)], cwd=root, env=dict(os.environ, PYTHONPATH=root), capture_output=True, text=True,
                       timeout=100)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "reported 5" in r.stdout


def test_a_length_beyond_the_cache_is_reported():
    """Single tokens whose length is already at the end, or beyond it: the last rows' answer, the length stays at the end, and a report."""
    from fastkv_amd import ops
    from fastkv_amd._lib import FASTKV_EOVERFLOW, FastKVNativeError
    q, k, v = (torch.randn(2, h, r, 64, device="cuda").half() for h, r in ((4, 1), (2, 30), (2, 30)))
    at = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")            # noqa: E731
    want = ops.decode_window_attention(q, k, v, at([29, 4]), 0.125, window=9, advance=False)
    for lens in ([30, 4], [2000, 4]):
        n = at(lens)
        assert torch.equal(want, ops.decode_window_attention(q, k, v, n, 0.125, window=9))
        assert n.tolist() == [30, 5]
        with pytest.raises(FastKVNativeError) as e:
            ops.raise_if_aborted()
        assert e.value.code == FASTKV_EOVERFLOW
