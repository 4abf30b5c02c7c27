"""The append with one length per request, and whole steps of it with the attention forms over a cache: ragged, idle and full requests, fp16
and bf16, eager and captured, against the rows that each request holds (attention against 64 bits: tests/attend_ref.py derives the
tolerance)."""
import pytest
import torch

from attend_ref import attend, check, prefix_rows, window_rows

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def rand(g, *shape, dtype):
    return torch.randn(*shape, generator=g).to(dtype)


def lengths(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def expected(slab, new, lens):
    """The slab [B,Hkv,rows,D] after the append: idle requests keep theirs, a full one's last row goes."""
    out = slab.clone()
    for b, n in enumerate(lens):
        if n >= 0:
            out[b, :, min(n, slab.shape[2] - 1)] = new[b, :, 0]
    return out


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_each_request_has_its_own_row(D, dtype):
    """The slabs lie inside larger tensors: nothing in front of them or behind them changes."""
    from fastkv_amd import ops
    g = torch.Generator().manual_seed(D)
    B, Hkv, rows = 6, 3, 20
    lens = [7, -1, 0, 19, 25, -2 ** 31]
    wide = [rand(g, B + 2, Hkv, rows, D, dtype=dtype) for _ in range(2)]
    new = [rand(g, B, 1, Hkv, D, dtype=dtype).transpose(1, 2) for _ in range(2)]
    dev = [w.cuda() for w in wide]
    n = lengths(lens)
    ops.decode_append(dev[0][1:-1], dev[1][1:-1], new[0].cuda(), new[1].cuda(), n)
    for w, d, x in zip(wide, dev, new):
        w[1:-1] = expected(w[1:-1], x, lens)
        assert torch.equal(d.cpu(), w)
    assert n.tolist() == lens


def test_one_length_for_all_is_as_before_and_an_idle_one_stores_nothing():
    from fastkv_amd import ops
    g = torch.Generator().manual_seed(1)
    slab, new = rand(g, 3, 2, 9, 64, dtype=F16), rand(g, 3, 2, 1, 64, dtype=F16)
    for n in (0, 4, 8, 100, -1):
        k, v = slab.cuda(), slab.cuda()
        ops.decode_append(k, v, new.cuda(), new.cuda(), lengths([n]))
        want = expected(slab, new, [n] * 3)
        assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), want)


@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 64), (BF16, 256)])
@pytest.mark.parametrize("form", ["window", "prefix"])
def test_steps_of_a_ragged_batch_eager_and_captured(form, dtype, D):
    """Steps of append + attention over requests of different lengths, one idle and one that runs into its slab's end."""
    from fastkv_amd import ops
    B, H, Hkv, rows, P, steps, window, sinks = 4, 8, 2, 90, 150, 4, 30, 3
    lens = [0, 61, -1, rows - 2]
    g = torch.Generator().manual_seed(D)
    k0, v0 = rand(g, B, Hkv, rows, D, dtype=dtype), rand(g, B, Hkv, rows, D, dtype=dtype)
    kp, vp = rand(g, Hkv, P, D, dtype=dtype), rand(g, Hkv, P, D, dtype=dtype)
    qs = [rand(g, B, 1, H, D, dtype=dtype).transpose(1, 2) for _ in range(steps)]
    ks, vs = ([rand(g, B, 1, Hkv, D, dtype=dtype).transpose(1, 2) for _ in range(steps)] for _ in range(2))
    dp = (kp.cuda(), vp.cuda())

    def step(s):
        ops.decode_append(s["k"], s["v"], s["kn"], s["vn"], s["n"])
        if form == "window":
            return ops.decode_window_attention(s["q"], s["k"], s["v"], s["n"], D ** -0.5, window=window, sinks=sinks)
        return ops.decode_shared_prefix_attention(s["q"], *dp, s["k"], s["v"], s["n"], D ** -0.5)

    def begin():
        return dict(k=k0.cuda(), v=v0.cuda(), n=lengths(lens), q=qs[0].cuda(), kn=ks[0].cuda(), vn=vs[0].cuda())

    def feed(s, i):
        for name, x in (("q", qs), ("kn", ks), ("vn", vs)):
            s[name].copy_(x[i].cuda())

    eager, captured = begin(), begin()
    graph, out = torch.cuda.CUDAGraph(), None
    k, v, now = k0.clone(), v0.clone(), list(lens)
    for i in range(steps):
        feed(eager, i)
        got = step(eager)
        k, v = expected(k, ks[i], now), expected(v, vs[i], now)
        assert torch.equal(eager["k"].cpu(), k) and torch.equal(eager["v"].cpu(), v)
        if form == "window":
            rows_of = window_rows(k.double(), v.double(), now, 1, window, sinks, Hkv, H)
        else:
            rows_of = prefix_rows(kp.double(), vp.double(), k.double(), v.double(), now, 1, Hkv, H)
        check(got, *attend(qs[i], rows_of, D ** -0.5))
        now = [n if n < 0 else min(n + 1, rows) for n in now]
        assert eager["n"].tolist() == now
        feed(captured, i)
        if i == 1:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.graph(graph, stream=side):
                out = step(captured)
            torch.cuda.current_stream().wait_stream(side)
        if i == 0:
            step(captured)
        else:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, got)
        assert torch.equal(captured["k"], eager["k"]) and torch.equal(captured["n"], eager["n"])
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError):                             # the full request said so
        ops.raise_if_aborted()
