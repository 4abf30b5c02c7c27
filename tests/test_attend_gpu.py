"""Attention with a sliding window and sinks, and over a shared prefix (csrc/attend.hip), against their plain 64-bit forms
(tests/attend_ref.py derives the tolerance)."""
import pytest
import torch

from attend_ref import attend, check, prefix_rows, window_rows

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def make(seed, B, H, Hkv, D, T, rows, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(B, T, H, D, generator=g) * scale).to(dtype).transpose(1, 2)
    k = (torch.randn(B, Hkv, rows, D, generator=g) * scale).to(dtype)
    v = torch.randn(B, Hkv, rows, D, generator=g).to(dtype)
    return q, k, v


def dev_lens(lens):
    return torch.tensor(lens, dtype=torch.int32, device="cuda")


WINDOW = [
    # B, H, Hkv, D, T, rows, window, sinks, dtype, lens (None: the last T rows)
    (1, 4, 1, 128, 1, 1, None, 0, F16, [0]),                  # one row
    (1, 4, 1, 128, 1, 70, 1, 0, F16, [63]),                   # a window of one
    (2, 8, 8, 64, 1, 300, 64, 4, BF16, [299, 17]),            # single tokens, ragged, one cache shorter than the window
    (3, 8, 1, 128, 1, 500, 100, 130, F16, [499, 0, 250]),     # more sinks than window; G = 8
    (2, 6, 2, 256, 1, 200, 33, 5, BF16, [150, 40]),           # G = 3, head_dim 256
    (1, 32, 2, 64, 3, 700, 200, 4, F16, [600]),               # G = 16, 48 rows
    (1, 4, 4, 128, 32, 90, None, 0, F16, None),               # 32 rows of one head, cache in front
    (2, 8, 2, 128, 33, 33, 7, 2, BF16, None),                 # a whole prompt, odd length, narrow window
    (1, 8, 8, 64, 129, 129, 64, 1, F16, None),                # one row more than a workgroup holds
    (1, 12, 4, 128, 100, 260, 31, 3, F16, [90]),              # G = 3: heads straddle the waves
    (2, 4, 2, 256, 70, 200, 50, 70, BF16, [130, 3]),          # head_dim 256, sinks inside and in front of the window
    (1, 5, 1, 64, 64, 400, 100, 0, F16, [300]),               # G = 5
    (1, 4, 1, 128, 20, 12, 5, 1, F16, None),                  # more queries than rows: the first eight see nothing
    (3, 4, 2, 64, 40, 100, 16, 2, BF16, [-10, -40, 55]),      # left padding, a request of padding only
    (2, 4, 2, 128, 1, 100, 16, 2, F16, [-1, 99]),             # an idle request
    (2, 4, 2, 128, 4, 100, 16, 2, F16, [2000, 3]),            # a length beyond the cache: its last rows
]


@pytest.mark.parametrize("B,H,Hkv,D,T,rows,window,sinks,dtype,lens", WINDOW)
def test_window_attention(B, H, Hkv, D, T, rows, window, sinks, dtype, lens):
    from fastkv_amd import ops
    q, k, v = make(B * 7 + T, B, H, Hkv, D, T, rows, dtype)
    scaling = D ** -0.5
    got = ops.window_attention(q.cuda(), k.cuda(), v.cuda(), window=window, sinks=sinks, len_dev=dev_lens(lens) if lens else None)
    ref, bound = attend(q, window_rows(k.double(), v.double(), lens or [rows - T] * B, T, window, sinks, Hkv, H), scaling)
    assert got.shape == (B, T, H * D) and got.dtype == dtype
    check(got, ref, bound)
    if T == 1:                                                # the single-token form is the same call, and moves the lengths on
        n = dev_lens(lens)
        two = ops.decode_window_attention(q.cuda(), k.cuda(), v.cuda(), n, scaling, window=window, sinks=sinks)
        check(two, ref, bound)
        assert n.tolist() == [x + 1 if 0 <= x < rows else min(x, rows) for x in lens]
        if max(lens) >= rows:
            with pytest.raises(RuntimeError):
                torch.cuda.synchronize()
                ops.raise_if_aborted()


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16), (128, F16), (256, F16)])
@pytest.mark.parametrize("T", [1, 20, 200])
def test_rows_that_nothing_sees_may_hold_anything(D, dtype, T):
    """Infinities and NaN behind the cache's end, in front of the window, and -- for the queries that do not see them -- between rows that others
    see: every query's result is that of the rows it sees alone."""
    from fastkv_amd import ops
    B, H, Hkv, rows, window, sinks = 2, 4, 2, 330, 40, 3
    q, k, v = make(T + D, B, H, Hkv, D, T, rows, dtype)
    lens = [90, 57]
    for b in range(B):
        for j in [rows - 1, lens[b] + T]:                      # behind the end
            if j >= lens[b] + T:
                k[b, :, j:] = float("nan")
                v[b, :, j:] = float("inf")
        k[b, :, sinks:lens[b] - window + 1] = float("inf")     # between the sinks and the first query's window
        v[b, :, sinks:lens[b] - window + 1] = float("nan")
    if T > 1:                                                  # seen by some queries of a tile only
        v[0, 0, lens[0] + T // 2, 5] = float("nan")
        v[1, 1, lens[1] + T // 3] = float("inf")
        v[0, 1, lens[0] + T - 1, 1] = -float("inf")
        k[1, 0, lens[1] + T // 2, 0] = float("nan")
    got = ops.window_attention(q.cuda(), k.cuda(), v.cuda(), window=window, sinks=sinks, len_dev=dev_lens(lens))
    ref, bound = attend(q, window_rows(k.double(), v.double(), lens, T, window, sinks, Hkv, H), D ** -0.5)
    assert torch.isfinite(ref).any()
    check(got, ref, bound)


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, F16), (256, BF16)])
@pytest.mark.parametrize("T", [9, 300])
def test_infinities_in_many_tiles(D, dtype, T):
    """Infinities and NaN in V rows of several partly seen tiles, in front of them and behind them, while the running maximum moves: the other
    dims of their pieces keep their values, and rows that do not see them stay finite."""
    from fastkv_amd import ops
    H, Hkv, n, window = 4, 2, 700, 260
    rows = n + T
    q, k, v = make(D + T, 1, H, Hkv, D, T, rows, dtype)
    k *= torch.linspace(0.2, 2.5, rows).to(dtype)[None, None, :, None]
    for i, j in enumerate(range(n - window - 3, rows, 37)):
        v[0, i % Hkv, j, (i * 11) % D] = [float("inf"), -float("inf"), float("nan")][i % 3]
    v[0, 0, 2, 3] = float("inf")                               # a sink
    v[0, 1, rows - 1] = float("nan")                           # a whole row, the last query's alone
    for sinks in (0, 4):
        got = ops.window_attention(q.cuda(), k.cuda(), v.cuda(), window=window, sinks=sinks)
        ref, bound = attend(q, window_rows(k.double(), v.double(), [n], T, window, sinks, Hkv, H), D ** -0.5)
        assert torch.isfinite(ref).any() and not torch.isfinite(ref).all()
        check(got, ref, bound)


def test_one_strong_key_among_many_weak_ones():
    """Thousands of keys 2^-15 of the strongest: each p is small for 16 bits, together they weigh as much as the strong one."""
    from fastkv_amd import ops
    D, rows = 64, 20000
    for dtype in (F16, BF16):
        q = torch.zeros(1, 1, 1, D, dtype=dtype)
        k = torch.zeros(1, 1, rows, D, dtype=dtype)
        q[..., 0], k[0, 0, 123, 0] = 1, 10.25                  # exp(-10.25) = 2^-14.8
        v = torch.randn(1, 1, rows, D, generator=torch.Generator().manual_seed(2)).to(dtype) + 1
        got = ops.window_attention(q.cuda(), k.cuda(), v.cuda(), scaling=1.0)
        ref, bound = attend(q, window_rows(k.double(), v.double(), [rows - 1], 1, None, 0, 1, 1), 1.0)
        check(got, ref, bound)


def test_growing_scores_and_large_ones():
    """Scores that grow along the keys (the running maximum moves in every tile) and spread over hundreds of powers of two."""
    from fastkv_amd import ops
    for dtype in (F16, BF16):
        q, k, v = make(5, 1, 4, 2, 64, 150, 600, dtype)
        k *= torch.linspace(0.1, 12, 600).to(dtype)[None, None, :, None]
        got = ops.window_attention(q.cuda(), k.cuda(), v.cuda(), window=500, sinks=2, scaling=0.5)
        ref, bound = attend(q, window_rows(k.double(), v.double(), [450], 150, 500, 2, 2, 4), 0.5)
        check(got, ref, bound)


def test_infinite_scores_follow_the_formula():
    from fastkv_amd import ops
    q, k, v = make(8, 1, 2, 1, 64, 1, 80, F16)
    k[0, 0, 40] = float("inf")
    got = ops.window_attention(q.cuda(), k.cuda(), v.cuda())
    assert torch.isnan(got).all()                              # inf - inf
    k[0, 0, 40] = 1
    q[0, 1] = float("nan")
    got = ops.window_attention(q.cuda(), k.cuda(), v.cuda())
    assert torch.isnan(got[..., 64:]).all() and torch.isfinite(got[..., :64]).all()


def test_window_attention_takes_the_strides_it_documents():
    from fastkv_amd import ops
    B, H, Hkv, D, T, rows = 2, 8, 2, 128, 45, 200
    q, k, v = make(3, B, H, Hkv, D, T, rows, F16)
    want = ops.window_attention(q.cuda(), k.cuda(), v.cuda(), window=60, sinks=4)
    q2 = q.contiguous().cuda()                                                              # [B,H,T,D] storage
    k2 = k.transpose(1, 2).contiguous().cuda().transpose(1, 2)                              # [B,rows,Hkv,D] storage
    wide = torch.full((B, Hkv, rows + 9, 2 * D), float("nan"), dtype=F16, device="cuda")     # a part of a wider slab
    wide[:, :, 4:rows + 4, D:] = v.cuda()
    assert torch.equal(want, ops.window_attention(q2, k2, wide[:, :, 4:rows + 4, D:], window=60, sinks=4))
    q3 = torch.empty(B, T, 3 * H, D, dtype=F16, device="cuda")                               # queries inside a fused projection
    q3[:, :, H:2 * H] = q.transpose(1, 2).cuda()
    assert torch.equal(want, ops.window_attention(q3[:, :, H:2 * H].transpose(1, 2), k.cuda(), v.cuda(), window=60, sinks=4))
    # one head for the whole batch: a stride of zero
    k4, v4 = k[:1, :1].cuda().expand(B, Hkv, rows, D), v[:1, :1].cuda().expand(B, Hkv, rows, D)
    assert torch.equal(ops.window_attention(q2, k4, v4, window=60), ops.window_attention(q2, k4.contiguous(), v4.contiguous(), window=60))


PREFIX = [
    # B, H, Hkv, D, T, P, rows, dtype, lens
    (1, 4, 1, 128, 1, 1, 8, F16, [0]),
    (3, 8, 2, 128, 1, 200, 40, F16, [0, 39, 7]),              # 12 rows: one wave's block
    (16, 8, 2, 64, 1, 333, 20, BF16, list(range(16))),        # 64 rows
    (40, 8, 1, 128, 1, 130, 9, F16, [i % 9 for i in range(40)]),   # 320 rows, G = 8: several row tiles
    (2, 6, 2, 256, 1, 100, 30, BF16, [29, 3]),                # G = 3, head_dim 256
    (4, 4, 2, 64, 17, 150, 70, F16, [0, 10, 53, 2]),          # questions of 17 tokens
    (2, 8, 2, 128, 40, 300, 90, BF16, [0, 50]),               # 160 rows per request: no packing over requests
    (1, 8, 8, 64, 130, 64, 130, F16, [0]),
    (3, 4, 2, 128, 1, 100, 16, F16, [-1, 5, 15]),             # an idle request
    (2, 4, 1, 128, 6, 90, 64, BF16, [-3, 30]),                # left padding
    (2, 4, 1, 64, 40, 90, 64, F16, [-20, 24]),
    (2, 8, 2, 128, 1, 150, 3500, F16, [3490, 100]),           # own rows far longer than the prefix: cut as well
    (2, 8, 2, 64, 5, 40, 1900, BF16, [1800, 3]),
]


@pytest.mark.parametrize("B,H,Hkv,D,T,P,rows,dtype,lens", PREFIX)
def test_shared_prefix_attention(B, H, Hkv, D, T, P, rows, dtype, lens):
    from fastkv_amd import ops
    q, k, v = make(B + T, B, H, Hkv, D, T, rows, dtype)
    _, kp, vp = make(B + T + 1, 1, H, Hkv, D, 1, P, dtype)
    for b in range(B):                                         # nobody reads rows behind a request's own end
        k[b, :, max(0, lens[b] + T):] = float("nan")
        v[b, :, max(0, lens[b] + T):] = float("nan")
    n = dev_lens(lens)
    args = (q.cuda(), kp.cuda(), vp.cuda(), k.cuda(), v.cuda())
    got = ops.decode_shared_prefix_attention(*args, n, D ** -0.5, advance=False)
    ref, bound = attend(q, prefix_rows(kp[0].double(), vp[0].double(), k.double(), v.double(), lens, T, Hkv, H), D ** -0.5)
    check(got, ref, bound)
    assert n.tolist() == lens
    two = ops.decode_shared_prefix_attention(args[0], kp[0].cuda(), vp[0].cuda(), *args[3:], n, D ** -0.5)
    check(two, ref, bound)
    assert n.tolist() == [x + T if x >= 0 else x for x in lens]


def test_one_length_for_all_and_the_full_cache():
    from fastkv_amd import ops
    from fastkv_amd._lib import FASTKV_EOVERFLOW, FastKVNativeError
    q, k, v = make(1, 3, 4, 2, 64, 1, 20, F16)
    args = (q.cuda(), k.cuda(), v.cuda())
    n = dev_lens([18])
    each = ops.decode_window_attention(*args, dev_lens([18, 18, 18]), 0.125, window=7, sinks=1, advance=False)
    assert torch.equal(each, ops.decode_window_attention(*args, n, 0.125, window=7, sinks=1))
    assert n.tolist() == [19]
    ops.decode_window_attention(*args, n, 0.125, window=7, sinks=1)
    assert n.tolist() == [20]
    torch.cuda.synchronize()
    ops.raise_if_aborted()
    ops.decode_window_attention(*args, n, 0.125, window=7, sinks=1)      # full: attends as at row 19, stays, and says so
    torch.cuda.synchronize()
    assert n.tolist() == [20]
    with pytest.raises(FastKVNativeError) as e:
        ops.raise_if_aborted()
    assert e.value.code == FASTKV_EOVERFLOW


def test_offsets_beyond_32_bits():
    """A slab whose rows lie more than 2^32 bytes (and elements of 2^31) apart from its base."""
    from fastkv_amd import ops
    D, rows, step = 128, 40, 1 << 27                           # 40 rows, 2^28 bytes apart: 10 GiB each
    big = torch.empty((rows - 1) * step + D, dtype=F16, device="cuda")
    k = big.as_strided((1, 1, rows, D), (0, 0, step, 1))
    q, ks, vs = make(4, 1, 4, 1, D, 5, rows, F16)
    k.copy_(ks)
    want = ops.window_attention(q.cuda(), ks.cuda(), vs.cuda(), window=11, sinks=2)
    assert torch.equal(want, ops.window_attention(q.cuda(), k, vs.cuda(), window=11, sinks=2))
    k.copy_(vs)
    assert torch.equal(want, ops.window_attention(q.cuda(), ks.cuda(), k, window=11, sinks=2))


def test_captured_and_replayed_with_eager_calls_between():
    """Two graphs of the same call, captured on one stream, replayed in turn (and one beside an eager call on another stream): nothing is
    shared between them."""
    from fastkv_amd import ops
    B, H, Hkv, D, P, rows = 4, 8, 2, 128, 700, 64
    q, k, v = (t.cuda() for t in make(1, B, H, Hkv, D, 1, rows, F16))
    _, kp, vp = (t.cuda() for t in make(2, 1, H, Hkv, D, 1, P, F16))
    lens = [3, 40, 0, 17]

    def step(q, n):
        a = ops.decode_shared_prefix_attention(q, kp, vp, k, v, n, 0.1)
        return a, ops.decode_window_attention(q, k, v, n, 0.1, window=9, sinks=2, advance=False)

    qs = [q, q.flip(0).contiguous()]
    ns = [dev_lens(lens), dev_lens(lens)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for i in range(2):
        step(qs[i], dev_lens(lens))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(step(qs[i], ns[i]))
        graphs.append(g)
    torch.cuda.current_stream().wait_stream(side)
    other = torch.cuda.Stream()
    for r in range(4):
        want = [step(qs[i], dev_lens([x + r for x in lens])) for i in range(2)]
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
            extra = step(qs[0], dev_lens([x + r for x in lens]))
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i][0], want[i][0]) and torch.equal(outs[i][1], want[i][1])
            assert ns[i].tolist() == [x + r + 1 for x in lens]
        assert torch.equal(extra[0], want[0][0]) and torch.equal(extra[1], want[0][1])


def test_the_same_call_gives_the_same_bits():
    from fastkv_amd import ops
    q, k, v = (t.cuda() for t in make(1, 2, 8, 2, 128, 1, 4000, BF16))
    n = dev_lens([3999, 2000])
    first = ops.decode_window_attention(q, k, v, n, 0.09, window=1500, sinks=4, advance=False)
    for _ in range(5):
        assert torch.equal(first, ops.decode_window_attention(q, k, v, n, 0.09, window=1500, sinks=4, advance=False))


def test_wide_window_agrees_with_the_dense_decode():
    """Beside its sibling: a window as long as the cache is decode_attention."""
    from fastkv_amd import ops
    q, k, v = (t.cuda() for t in make(6, 1, 32, 8, 128, 1, 2304, F16))
    n1, n2 = dev_lens([2100]), dev_lens([2100])
    a = ops.decode_attention(q, k, v, n1, 128 ** -0.5).float()
    b = ops.decode_window_attention(q, k, v, n2, 128 ** -0.5).float()
    assert float((a - b).abs().max()) <= 2e-3 * float(a.abs().max()) + 1e-3
    assert n1.tolist() == n2.tolist() == [2101]


def test_front_end_refusals():
    from fastkv_amd import ops
    q, k, v = (t.cuda() for t in make(1, 2, 4, 2, 64, 1, 20, F16))
    n = dev_lens([3, 4])
    with pytest.raises(TypeError, match="fp16 or bf16"):
        ops.window_attention(q.float(), k, v)
    with pytest.raises(TypeError, match="one type"):
        ops.window_attention(q, k, v.bfloat16())
    for bad in (q[:1], q[..., :32], q[:, :3], q[0]):
        with pytest.raises(ValueError, match="expected q"):
            ops.window_attention(bad, k, v)
    with pytest.raises(ValueError, match="head_dim stride"):
        ops.window_attention(q, k.transpose(2, 3).contiguous().transpose(2, 3), v)
    for bad in (n.long(), n[:, None], dev_lens([1, 2, 3])):
        with pytest.raises(ValueError, match="len_dev"):
            ops.window_attention(q, k, v, len_dev=bad)
    with pytest.raises(RuntimeError, match="one ROCm device"):
        ops.window_attention(q, k, v, len_dev=n.cpu())
    for kw in (dict(window=0), dict(window=-3), dict(sinks=-1)):
        with pytest.raises(ValueError, match="window >= 1"):
            ops.window_attention(q, k, v, **kw)
    with pytest.raises(ValueError, match="no rows"):
        ops.window_attention(q, k[:, :, :0], v[:, :, :0])
    with pytest.raises(RuntimeError, match="no backward"):
        ops.window_attention(q.clone().requires_grad_(), k, v)
    with torch.no_grad():
        ops.window_attention(q.clone().requires_grad_(), k, v)
    with pytest.raises(ValueError, match="len_dev expected"):
        ops.decode_window_attention(q, k, v, None, 0.1)
    with pytest.raises(ValueError, match="expected prefixes"):
        ops.decode_shared_prefix_attention(q, k[0, :, :0], v[0, :, :0], k, v, n, 0.1)
    with pytest.raises(ValueError, match="new tokens in slabs"):
        ops.decode_shared_prefix_attention(torch.zeros(2, 4, 30, 64, dtype=F16, device="cuda"), k[0], v[0], k, v, n, 0.1)
    assert ops.window_attention(q[:0], k[:0], v[:0]).shape == (0, 1, 256)
    assert ops.window_attention(q[:, :, :0], k, v).shape == (2, 0, 256)


def test_on_another_stream_than_the_tensors():
    from fastkv_amd import ops
    q, k, v = (t.cuda() for t in make(1, 2, 8, 2, 128, 1, 3000, F16))
    n = dev_lens([2500, 100])
    want = ops.decode_window_attention(q, k, v, n, 0.1, window=900, sinks=4, advance=False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [ops.decode_window_attention(q, k, v, n, 0.1, window=900, sinks=4, advance=False) for _ in range(8)]
    here = [ops.decode_window_attention(q, k, v, n, 0.1, window=900, sinks=4, advance=False) for _ in range(8)]
    torch.cuda.synchronize()
    assert all(torch.equal(want, x) for x in got + here)


def test_idle_lengths_strides_of_single_extents_and_many_heads_per_kv_head():
    from fastkv_amd import ops
    q, k, v = make(2, 3, 4, 2, 64, 2, 30, F16)
    lens = [-2 ** 31, 7, 2 ** 31 - 1]                               # idle for good, in use, beyond the cache
    got = ops.window_attention(q.cuda(), k.cuda(), v.cuda(), window=5, sinks=1, len_dev=dev_lens(lens))
    ref, bound = attend(q, window_rows(k.double(), v.double(), [-2, 7, 28], 2, 5, 1, 2, 4), 64 ** -0.5)
    check(got, ref, bound)
    # extents of one may have any stride
    one = torch.randn(64, dtype=F16, device="cuda").as_strided((1, 1, 1, 64), (3, 5, 7, 1))
    assert torch.equal(ops.window_attention(one, one, one)[0, 0], one[0, 0, 0])
    # 40 query heads on one KV head: two row tiles for a single token
    q, k, v = make(3, 2, 40, 1, 128, 1, 90, BF16)
    got = ops.decode_window_attention(q.cuda(), k.cuda(), v.cuda(), dev_lens([89, 30]), 0.09, window=33, sinks=2, advance=False)
    ref, bound = attend(q, window_rows(k.double(), v.double(), [89, 30], 1, 33, 2, 1, 40), 0.09)
    check(got, ref, bound)


@pytest.mark.parametrize("H,Hkv,window", [(6, 3, None), (8, 1, None), (8, 8, 150)])
def test_longer_prompts_against_sdpa_in_fp32(H, Hkv, window):
    """Enough row tiles for every die, in runs or whole heads: each row of the output is where it belongs."""
    from fastkv_amd import ops
    T, D = 2111, 64
    q, k, v = (t.cuda() for t in make(H, 1, H, Hkv, D, T, T, F16))
    got = ops.window_attention(q, k, v, window=window, sinks=2).float().view(T, H, D)
    kk, vv = (t.float().repeat_interleave(H // Hkv, 1)[0] for t in (k, v))
    i, j = torch.arange(T, device="cuda")[:, None], torch.arange(T, device="cuda")[None]
    ok = (j <= i) & ((j < 2) | (j > i - (window or T)))
    s = (q[0].float() @ kk.transpose(-1, -2).contiguous()) * D ** -0.5
    want = (torch.softmax(s.masked_fill(~ok, -float("inf")), -1) @ vv).transpose(0, 1)
    A = float(vv.abs().max())                                        # no less than any sum p |v|: two roundings of half a step of it
    assert float((got - want).abs().max()) <= 2 ** -10 * A


def test_prefix_inside_a_longer_slab_of_another_batch():
    """The prefix as a view of a cache slab (rows of another stride than the requests' own), for few and for many rows per request."""
    from fastkv_amd import ops
    H, Hkv, D, P = 8, 2, 128, 170
    slab_k, slab_v = (torch.full((1, Hkv, 300, D + 64), float("nan"), dtype=F16) for _ in range(2))
    for T in (1, 5, 60):
        q, k, v = make(T, 2, H, Hkv, D, T, 80, F16)
        _, kp, vp = make(T + 1, 1, H, Hkv, D, 1, P, F16)
        slab_k[:, :, 20:20 + P, :D], slab_v[:, :, 20:20 + P, :D] = kp, vp
        sk, sv = slab_k.cuda(), slab_v.cuda()
        got = ops.decode_shared_prefix_attention(q.cuda(), sk[:, :, 20:20 + P, :D], sv[0, :, 20:20 + P, :D][None], k.cuda(), v.cuda(), dev_lens([3, 20]), 0.1,
                                                 advance=False)
        ref, bound = attend(q, prefix_rows(kp[0].double(), vp[0].double(), k.double(), v.double(), [3, 20], T, Hkv, H), 0.1)
        check(got, ref, bound)


def test_together_as_a_step_uses_them_captured():
    """One document, four requests: the questions' own prefill, then captured single-token steps -- append, attention over prefix and own rows, penalties,
    greedy choice -- against the same steps run eagerly."""
    from fastkv_amd import ops
    B, H, Hkv, D, P, rows, T, V, steps = 4, 8, 2, 64, 300, 64, 9, 512, 6
    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=F16)                      # noqa: E731
    kp, vp, emb, wq, wk, wv, out_w = rnd(Hkv, P, D), rnd(Hkv, P, D), rnd(V, 64), rnd(64, H * D) / 8, rnd(64, Hkv * D) / 8, rnd(64, Hkv * D) / 8, rnd(H * D, V) / 22
    question = torch.randint(0, V, (B, T), generator=g, device="cuda")

    def begin():
        s = dict(k=torch.full((B, Hkv, rows, D), float("nan"), dtype=F16, device="cuda"), n=dev_lens([0]), tok=torch.zeros(B, 1, dtype=torch.int64, device="cuda"),
                 hist=torch.zeros(B, rows, dtype=torch.int64, device="cuda"), nt=dev_lens([T] * B), np=dev_lens([T] * B),
                 scratch=ops.new_greedy_scratch(kp.device, B), rep=torch.full((1,), 1.3, device="cuda"), freq=torch.full((1,), 0.5, device="cuda"))
        s["v"] = s["k"].clone()
        s["hist"][:, :T] = question
        x = emb[question]
        heads = lambda w, h: (x @ w).view(B, T, h, D).transpose(1, 2)                            # noqa: E731
        s["k"][:, :, :T], s["v"][:, :, :T] = heads(wk, Hkv), heads(wv, Hkv)
        a = ops.decode_shared_prefix_attention(heads(wq, H), kp, vp, s["k"], s["v"], s["n"], D ** -0.5)
        choose(s, a[:, -1:])
        return s

    def choose(s, a):
        logits = (a @ out_w).view(B, V)
        x = ops.decode_penalties(logits, s["hist"], s["nt"], s["np"], repetition=s["rep"], frequency=s["freq"])
        ops.decode_greedy(x[:, None], s["scratch"], s["tok"])
        s["hist"].scatter_(1, s["nt"].long()[:, None], s["tok"])
        s["nt"].add_(1)

    def step(s):
        x = emb[s["tok"][:, 0]][:, None]
        heads = lambda w, h: (x @ w).view(B, 1, h, D).transpose(1, 2)                            # noqa: E731
        ops.decode_append(s["k"], s["v"], heads(wk, Hkv), heads(wv, Hkv), s["n"])
        choose(s, ops.decode_shared_prefix_attention(heads(wq, H), kp, vp, s["k"], s["v"], s["n"], D ** -0.5))

    eager = begin()
    for _ in range(steps):
        step(eager)
    s = begin()
    step(s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(s)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(steps - 1):
        graph.replay()
        torch.cuda.synchronize()
        eager["k"].nan_to_num().sum()                                # the program's own work between the replays
    assert int(s["n"]) == int(eager["n"]) == T + steps
    assert torch.equal(s["hist"], eager["hist"]) and torch.equal(s["nt"], eager["nt"])
    assert len(set(s["hist"][0, T:T + steps + 1].tolist())) > 1
