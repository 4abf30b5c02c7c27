"""Penalties, biases and masks on a step's logits (csrc/penalties.hip) against the formula in 64 bits.

Tolerance: five fp32 operations of at most half a step (2^-24) of the largest intermediate value each, and the rounding to the logits'
type (half a step: 2^-11 fp16, 2^-8 bf16, 2^-24 fp32; fp16 subnormals 2^-25)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def formula(x, tokens, n, n0, rep, pres, freq, bias, allowed):
    """(result, bound) in fp64 on the CPU; every argument there, None where it is not given."""
    B, V = x.shape
    half = HALF[x.dtype]
    x = x.double()
    size = x.abs()
    for b in range(B):
        at = lambda t: None if t is None else t[b if t.shape[0] > 1 else 0]      # noqa: E731
        if tokens is not None:
            nb = tokens.shape[1] if n is None else min(int(at(n)), tokens.shape[1])
            ids = tokens[b, :max(0, nb)]
            first = 0 if n0 is None else int(at(n0))
            for v in set(ids.tolist()):
                if not 0 <= v < V:
                    continue
                if rep is not None:
                    r = float(at(rep))
                    x[b, v] = x[b, v] / r if x[b, v] > 0 else x[b, v] * r
                size[b, v] = max(float(size[b, v]), float(x[b, v].abs()))
                c = int((ids[max(0, first):] == v).sum())
                if freq is not None:
                    x[b, v] -= float(at(freq)) * c
                    size[b, v] += abs(float(at(freq)) * c)
                if pres is not None and c:
                    x[b, v] -= float(at(pres))
                    size[b, v] += abs(float(at(pres)))
        if bias is not None:
            row = bias if bias.dim() == 1 else bias[b if bias.shape[0] > 1 else 0]
            x[b] += row.double()
            size[b] += row.double().abs()
        if allowed is not None:
            words = allowed if allowed.dim() == 1 else allowed[b if allowed.shape[0] > 1 else 0]
            for v in range(V):
                if not int(words[v // 32]) >> (v % 32) & 1:
                    x[b, v] = -float("inf")
    return x, half * x.abs() + 5 * 2.0 ** -24 * size + (2.0 ** -25 if half == 2.0 ** -11 else 0.0)


def check(got, ref, bound):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    fine = torch.isfinite(ref)
    assert torch.equal(got[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)])
    assert bool(((got - ref).abs() <= bound)[fine].all()), float(((got - ref).abs() - bound)[fine].max())


def make(seed, B, V, L, dtype):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.rand(*s, generator=g)                                     # noqa: E731
    return dict(x=(torch.randn(B, V, generator=g) * 3).to(dtype), tokens=(r(B, L) ** 2 * V).long().clamp_(max=V - 1),
                n=torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32), n0=torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32),
                rep=1 + r(B) * 0.5, pres=r(B) - 0.5, freq=r(B) - 0.3, bias=torch.randn(B, V, generator=g),
                allowed=torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32), generator=g, dtype=torch.int32))


def call(ops, s, out=None):
    d = {k: v.cuda() if v is not None else None for k, v in s.items()}
    return ops.decode_penalties(d["x"], d["tokens"], d["n"], d["n0"], d["rep"], d["pres"], d["freq"], d["bias"], d["allowed"], out)


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("B,V,L", [(1, 1, 1), (1, 7, 3), (3, 33, 40), (2, 4096, 100), (5, 4099, 700), (2, 9000, 6000), (70, 520, 30), (1, 40000, 50)])
def test_all_of_it(B, V, L, dtype):
    from fastkv_amd import ops
    s = make(B * V + L, B, V, L, dtype)
    check(call(ops, s), *formula(**s))


@pytest.mark.parametrize("left", ["rep", "pres", "freq", "bias", "allowed", "n0", "n", None])
def test_each_part_alone(left):
    from fastkv_amd import ops
    s = make(4, 3, 500, 60, torch.float32)
    if left is None:                                              # nothing at all: the logits as they are
        s = {k: v if k == "x" else None for k, v in s.items()}
        assert torch.equal(call(ops, s).cpu(), s["x"])
        return
    keep = {"x", "tokens", left} | ({"freq", "n"} if left in ("n0", "n") else set())
    s = {k: v if k in keep else None for k, v in s.items()}
    check(call(ops, s), *formula(**s))


def test_shared_rows_and_single_values():
    from fastkv_amd import ops
    s = make(9, 4, 260, 50, torch.float16)
    for k in ("n", "n0", "rep", "pres", "freq", "bias", "allowed"):
        s[k] = s[k][:1]
    check(call(ops, s), *formula(**s))
    s["bias"], s["allowed"] = s["bias"][0], s["allowed"][0]
    check(call(ops, s), *formula(**s))


def test_ids_outside_the_vocabulary_and_lengths_outside_the_history():
    from fastkv_amd import ops
    s = make(2, 3, 100, 40, torch.float32)
    s["tokens"][:, ::3] = -1
    s["tokens"][:, 1::3] = torch.tensor([100, 2 ** 40, -2 ** 62])[:, None]
    s["n"] = torch.tensor([1000, -5, 40], dtype=torch.int32)
    s["n0"] = torch.tensor([-7, 3, 1000], dtype=torch.int32)
    check(call(ops, s), *formula(**s))


def test_a_row_with_nothing_allowed_and_special_logits():
    from fastkv_amd import ops
    for dtype in HALF:
        s = make(3, 3, 96, 20, dtype)
        s["x"][1, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), 0.0]).to(dtype)
        s["x"][2, 5] = torch.finfo(dtype).min
        s["rep"][2], s["pres"][2], s["freq"][2], s["bias"][2, 5] = 1, 0, 0, 0
        s["allowed"][0], s["allowed"][1], s["allowed"][2] = 0, -1, -1
        s["tokens"][1, :6] = torch.tensor([0, 1, 2, 3, 3, 3])
        s["n"][1], s["n0"][1] = 6, 1
        got = call(ops, s)
        check(got, *formula(**s))
        assert torch.isinf(got[0]).all()


def test_strides_and_in_place():
    from fastkv_amd import ops
    s = make(6, 3, 1000, 60, torch.float16)
    want = call(ops, s)
    for pad in (8, 3):                                            # 16-byte rows, and rows that are not
        wide = torch.full((3, 1000 + pad), float("nan"), dtype=torch.float16, device="cuda")
        wide[:, :1000] = s["x"].cuda()
        got = ops.decode_penalties(wide[:, :1000], s["tokens"].cuda(), s["n"].cuda(), s["n0"].cuda(), s["rep"].cuda(), s["pres"].cuda(),
                                   s["freq"].cuda(), s["bias"].cuda(), s["allowed"].cuda(), out=wide[:, :1000])
        assert got.data_ptr() == wide.data_ptr() and torch.equal(got, want) and torch.isnan(wide[:, 1000:]).all()
    odd = torch.zeros(3 * 1000 + 1, dtype=torch.float16, device="cuda")[1:].view(3, 1000)
    assert torch.equal(call(ops, s, out=odd), want)
    hist = torch.full((3, 90), 7, dtype=torch.int64)              # a history inside a longer log
    hist[:, 30:] = s["tokens"]
    assert torch.equal(ops.decode_penalties(s["x"].cuda(), hist.cuda()[:, 30:], s["n"].cuda(), s["n0"].cuda(), s["rep"].cuda(), s["pres"].cuda(),
                                            s["freq"].cuda(), s["bias"].cuda(), s["allowed"].cuda()), want)


def test_in_front_of_the_greedy_step_captured_and_replayed():
    """As a captured decode step uses it: penalties on the step's logits, the greedy token, and the history that grows on the device."""
    from fastkv_amd import ops
    V, L = 512, 40
    g = torch.Generator().manual_seed(11)
    logits = torch.randn(1, 1, V, generator=g).half().cuda()
    hist = torch.full((1, L), -1, dtype=torch.int64, device="cuda")
    hist[0, :3] = torch.tensor([5, 9, 5])
    n, n0 = torch.tensor([3], dtype=torch.int32, device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda")
    at = torch.zeros(1, dtype=torch.int64, device="cuda")
    freq, rep = torch.tensor([0.75], device="cuda"), torch.tensor([1.5], device="cuda")
    tok, scratch = torch.zeros(1, 1, dtype=torch.int64, device="cuda"), ops.new_greedy_scratch(logits.device, 1)

    def step():
        x = ops.decode_penalties(logits[:, -1], hist, n, n0, repetition=rep, frequency=freq)
        ops.decode_greedy(x[:, None], scratch, tok, None, hist[0, 3:], at)
        n.add_(1)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(20):
        graph.replay()
        torch.cuda.synchronize()
        logits.abs().sum()                                        # the program's own work between the replays
    ids = hist[0, 3:24].tolist()
    x0, said = logits[0, 0].double().cpu(), [5, 9, 5]
    for i, tok_i in enumerate(ids):
        x = x0.clone()
        for v in set(said):
            x[v] = x[v] / 1.5 if x[v] > 0 else x[v] * 1.5
            x[v] -= 0.75 * said[3:].count(v)
        x = x.half()
        assert int((x == x.max()).nonzero()[0]) == tok_i, i       # the first of equal ones
        said.append(tok_i)
    assert int(n) == 3 + 21 and len(set(ids)) > 3
