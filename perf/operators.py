"""The workloads of the operators beside the decode over a compressed cache: attention with a sliding window and sinks (prompts and single
tokens), attention of a batch over one shared prefix, and the penalties / biases / masks on a step's logits.

`own` False: the operators in their plain form (elementary torch operations in 32 bits, rounded once).  `own` True: the calls of
fastkv_amd.ops.  Head layouts are those of the repository's geometries (32 query heads on 8 KV heads of 128; 8 on 1; 64 and 256 as
head sizes of its operators), prompt and cache lengths those of its benchmarks."""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
WORDS = {"f16": 2, "bf16": 2, "f32": 4}


# ---------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # ---- a sliding window with sinks, prompts
        # a 32k prompt of the 8B geometry under a 4096-token window: the largest
        dict(op="window", name="prompt_32k", B=1, H=32, Hkv=8, D=128, T=32768, rows=32768, low=0, high=0, window=4096, sinks=4, dtype="f16"),
        # the same prompt length as most requests have
        dict(op="window", name="prompt_8k", B=1, H=32, Hkv=8, D=128, T=8192, rows=8192, low=0, high=0, window=4096, sinks=4, dtype="f16"),
        # a batch of short prompts of a small multi-head model, odd length, narrow window
        dict(op="window", name="short_prompts_odd", B=3, H=8, Hkv=8, D=64, T=1111, rows=1111, low=0, high=0, window=200, sinks=3, dtype="bf16"),
        # one chunk of a long prompt over what is cached already, requests of different lengths
        dict(op="window", name="chunk_over_cache", B=2, H=32, Hkv=8, D=128, T=512, rows=16384, low=9000, high=15800, window=4096, sinks=4,
             dtype="bf16"),
        # ---- the same, single tokens
        # one request whose cache has outgrown its window
        dict(op="window", name="token_one_request", B=1, H=32, Hkv=8, D=128, T=1, rows=5000, low=4800, high=4800, window=2048, sinks=4, dtype="f16"),
        # a serving batch with ragged caches
        dict(op="window", name="token_batch_32", B=32, H=32, Hkv=8, D=128, T=1, rows=16384, low=700, high=16000, window=4096, sinks=4, dtype="bf16"),
        # ---- a batch over one shared prefix
        # sixteen continuations of one prompt compressed to the constant budget
        dict(op="prefix", name="budget_16_requests", B=16, H=32, Hkv=8, D=128, T=1, P=2048, rows=256, low=1, high=200, dtype="f16"),
        # sixty-four requests on an uncompressed 32k document
        dict(op="prefix", name="document_64_requests", B=64, H=32, Hkv=8, D=128, T=1, P=32768, rows=512, low=10, high=500, dtype="f16"),
        # the questions themselves: 61 tokens each behind a document compressed by the published recipe
        dict(op="prefix", name="questions_of_61", B=8, H=32, Hkv=8, D=128, T=61, P=6553, rows=128, low=0, high=40, dtype="bf16"),
        # ---- a step's logits
        # one request with its whole history
        dict(op="penalties", name="one_row_128k", B=1, V=128256, L=2304, low=2304, high=2304, bias=0, mask=0, dtype="f16"),
        # a serving batch, everything in use
        dict(op="penalties", name="batch_64_all", B=64, V=131072, L=4096, low=16, high=4096, bias=2, mask=2, dtype="f32"),
        # a few rows under one grammar, a shared bias
        dict(op="penalties", name="grammar_5_rows", B=5, V=32000, L=700, low=5, high=700, bias=1, mask=1, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["window", "window", "token", "prefix", "penalties"])
    if op == "penalties":
        B, V, L = _log(rng, 1, 64), rng.choice([32000, 32768, 128256, 131072, 8 * rng.randint(64, 16000)]), _log(rng, 1, 8192)
        low = rng.randint(0, L)
        return dict(op=op, B=B, V=V, L=L, low=low, high=rng.randint(low, L), bias=rng.randint(0, 2), mask=rng.randint(0, 2),
                    dtype=rng.choice(["f16", "bf16", "f32"]))
    H, Hkv = rng.choice([(32, 8), (32, 8), (8, 8), (8, 1), (16, 8), (12, 4)])
    D = rng.choice([64, 128, 128, 128, 256])
    dtype = rng.choice(["f16", "bf16"])
    if op == "prefix":
        T = rng.choice([1, 1, 1, _log(rng, 2, 128)])
        B = _log(rng, 1, 64 if T == 1 else 8)
        rows = T + _log(rng, 1, 512)
        low = rng.randint(0, rows - T)
        return dict(op=op, B=B, H=H, Hkv=Hkv, D=D, T=T, P=_log(rng, 1, 32768 if T == 1 else 8192), rows=rows, low=low,
                    high=rng.randint(low, rows - T), dtype=dtype)
    if op == "token":
        B, rows = _log(rng, 1, 32), _log(rng, 2, 16384)
        low = rng.randint(0, rows - 1)
        return dict(op="window", B=B, H=H, Hkv=Hkv, D=D, T=1, rows=rows, low=low, high=rng.randint(low, rows - 1), window=_log(rng, 1, 8192),
                    sinks=rng.choice([0, 1, 4, 4, 16, 100]), dtype=dtype)
    T = _log(rng, 2, 8192)
    B = rng.randint(1, max(1, min(4, 8192 // T)))
    before = rng.choice([0, 0, _log(rng, 1, 8192)])
    low = rng.randint(0, before)
    return dict(op="window", B=B, H=H, Hkv=Hkv, D=D, T=T, rows=T + before, low=low, high=rng.randint(low, before), window=_log(rng, 16, 8192),
                sinks=rng.choice([0, 1, 4, 4, 64]), dtype=dtype)


# ---------------------------------------------------------------------------------------------------------------- the inputs
def _spread(case):
    """The requests' lengths, as whole numbers: evenly from `low` to `high`."""
    B, lo, hi = case["B"], case["low"], case["high"]
    return [hi if B == 1 else lo + (hi - lo) * b // (B - 1) for b in range(B)]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt, B = DTYPES[case["dtype"]], case["B"]
    order = torch.randperm(B, generator=torch.Generator().manual_seed(seed))
    lens = torch.tensor(_spread(case), dtype=torch.int32)[order].to(dev)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=dt)

    if case["op"] == "penalties":
        V, L = case["V"], case["L"]
        s = dict(logits=(torch.randn(B, V, generator=g, device=dev) * 3).to(dt), n_tokens=lens, n_prompt=lens // 2)
        s["tokens"] = (torch.rand(B, L, generator=g, device=dev) ** 3 * V).long().clamp_(max=V - 1)     # frequent tokens repeat
        s["repetition"] = 1 + torch.rand(B, generator=g, device=dev) * 0.5
        s["presence"] = torch.rand(B, generator=g, device=dev) - 0.25
        s["frequency"] = torch.rand(B, generator=g, device=dev) * 0.5
        s["bias"] = s["allowed"] = None
        if case["bias"]:                                                          # 1: one for the batch, 2: one per row
            s["bias"] = torch.randn(1 if case["bias"] == 1 else B, V, generator=g, device=dev)
        if case["mask"]:
            s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (1 if case["mask"] == 1 else B, (V + 31) // 32), generator=g, device=dev,
                                         dtype=torch.int32)
        return dict(case=case, **s)
    H, Hkv, D, T, rows = case["H"], case["Hkv"], case["D"], case["T"], case["rows"]
    # queries as the attention module has them: [B,T,H,D] storage seen as [B,H,T,D]; K / V: the cache's slabs, new rows written
    s = dict(q=rand(B, T, H, D).transpose(1, 2), k=rand(B, Hkv, rows, D), v=rand(B, Hkv, rows, D), lens=lens, scaling=D ** -0.5)
    if case["op"] == "prefix":
        s["kp"], s["vp"] = rand(1, Hkv, case["P"], D), rand(1, Hkv, case["P"], D)
    elif case["sinks"]:
        s["k"][:, :, :case["sinks"]] *= 1.5                                        # the first tokens draw attention
    return dict(case=case, **s)


# ---------------------------------------------------------------------------------------------------------------- the calls
def run(state):
    op = state["case"]["op"]
    return _penalties(state) if op == "penalties" else _prefix(state) if op == "prefix" else _window(state)


def _softmax_v(parts):
    """sum softmax(x) v over the concatenated (scores, values) parts; scores are overwritten."""
    m = torch.stack([x.amax(-1) for x, _ in parts]).amax(0)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m).unsqueeze(-1)
    e = [(x.sub_(m).exp_(), v) for x, v in parts]
    total = sum(x.sum(-1, keepdim=True) for x, _ in e)
    out = sum(torch.matmul(x, v) for x, v in e)
    return torch.where(total > 0, out / total, torch.zeros_like(out))


def _window(s):
    c, q = s["case"], s["q"]
    if own:
        from fastkv_amd import ops
        if c["T"] == 1:
            return ops.decode_window_attention(q, s["k"], s["v"], s["lens"], s["scaling"], window=c["window"], sinks=c["sinks"], advance=False)
        return ops.window_attention(q, s["k"], s["v"], window=c["window"], sinks=c["sinks"], scaling=s["scaling"], len_dev=s["lens"])
    B, H, Hkv, D, T, rows = (c[n] for n in ("B", "H", "Hkv", "D", "T", "rows"))
    G, W, dev = H // Hkv, min(c["window"], rows), q.device
    step = min(T, 512)                                       # queries of a block share one run of W + step - 1 rows
    nb, span = -(-T // step), W + step - 1
    p = s["lens"].long()[:, None, None] + torch.arange(nb * step, device=dev).view(1, nb, step)            # [B,nb,step]
    j = p[:, :, :1] - (W - 1) + torch.arange(span, device=dev)                                               # [B,nb,span]
    at = j.clamp(0, rows - 1)[:, None, :, :].expand(B, Hkv, nb, span)
    heads = torch.arange(Hkv, device=dev)[None, :, None, None]
    batch = torch.arange(B, device=dev)[:, None, None, None]
    k, v = s["k"][batch, heads, at].float(), s["v"][batch, heads, at].float()                               # [B,Hkv,nb,span,D]
    qs = torch.nn.functional.pad(q.float() * s["scaling"], (0, 0, 0, nb * step - T)).reshape(B, Hkv, G, nb, step, D)
    qs = qs.permute(0, 1, 3, 2, 4, 5).reshape(B, Hkv, nb, G * step, D)
    seen = (j[:, :, None, :] <= p[..., None]) & (j[:, :, None, :] > p[..., None] - W) & (j[:, :, None, :] >= min(c["sinks"], rows))
    x = torch.matmul(qs, k.transpose(-1, -2).contiguous())
    x.view(B, Hkv, nb, G, step, span).masked_fill_(~seen[:, None, :, None], -math.inf)
    parts = [(x, v)]
    n = min(c["sinks"], rows)
    if n:
        ks, vs = s["k"][:, :, None, :n].float(), s["v"][:, :, None, :n].float()
        x0 = torch.matmul(qs, ks.transpose(-1, -2).contiguous())
        early = torch.arange(n, device=dev) <= p[..., None]
        x0.view(B, Hkv, nb, G, step, n).masked_fill_(~early[:, None, :, None], -math.inf)
        parts.append((x0, vs))
    out = _softmax_v(parts).view(B, Hkv, nb, G, step, D).permute(0, 2, 4, 1, 3, 5).reshape(B, nb * step, H * D)
    return out[:, :T].to(q.dtype)


def _prefix(s):
    c, q = s["case"], s["q"]
    if own:
        from fastkv_amd import ops
        return ops.decode_shared_prefix_attention(q, s["kp"], s["vp"], s["k"], s["v"], s["lens"], s["scaling"], advance=False)
    B, H, Hkv, D, T, P, rows = (c[n] for n in ("B", "H", "Hkv", "D", "T", "P", "rows"))
    G, dev = H // Hkv, q.device
    qs = q.float().mul(s["scaling"]).reshape(B, Hkv, G, T, D)
    x = torch.matmul(qs.permute(1, 0, 2, 3, 4).reshape(Hkv, B * G * T, D), s["kp"][0].float().transpose(-1, -2).contiguous())
    x = x.view(Hkv, B, G, T, P).permute(1, 0, 2, 3, 4).reshape(B, Hkv, G * T, P)
    y = torch.matmul(qs.reshape(B, Hkv, G * T, D), s["k"].float().transpose(-1, -2).contiguous())
    p = s["lens"].long()[:, None] + torch.arange(T, device=dev)
    seen = torch.arange(rows, device=dev) <= p[..., None]                                                    # [B,T,rows]
    y.view(B, Hkv, G, T, rows).masked_fill_(~seen[:, None, None], -math.inf)
    out = _softmax_v([(x, s["vp"].float()), (y, s["v"].float())])
    return out.view(B, H, T, D).transpose(1, 2).reshape(B, T, H * D).to(q.dtype)


def _penalties(s):
    logits, tokens = s["logits"], s["tokens"]
    if own:
        from fastkv_amd import ops
        return ops.decode_penalties(logits, tokens, n_tokens=s["n_tokens"], n_prompt=s["n_prompt"], repetition=s["repetition"],
                                    presence=s["presence"], frequency=s["frequency"], bias=s["bias"], allowed=s["allowed"])
    B, V = logits.shape
    place = torch.arange(tokens.shape[1], device=logits.device)
    said = place < s["n_tokens"][:, None]
    again = said & (place >= s["n_prompt"][:, None])
    seen = torch.zeros(B, V, device=logits.device).scatter_add_(1, tokens, said.float()) > 0
    count = torch.zeros(B, V, device=logits.device).scatter_add_(1, tokens, again.float())
    x, rep = logits.float(), s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count
    x = torch.where(count > 0, x - s["presence"][:, None], x)
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["allowed"] is not None:
        bit = torch.arange(V, device=logits.device)
        x = torch.where((s["allowed"][:, bit // 32] >> (bit % 32)) & 1 == 1, x, -math.inf)
    return x.to(logits.dtype)


# ---------------------------------------------------------------------------------------------------------------- what a pass costs
def work(case):
    B, w = case["B"], WORDS[case["dtype"]]
    lens = _spread(case)
    if case["op"] == "penalties":
        V = case["V"]
        read = 2 * w * B * V + 8 * sum(lens) + 20 * B
        read += 4 * V * (0, 1, B)[case["bias"]] + 4 * ((V + 31) // 32) * (0, 1, B)[case["mask"]]
        return {"bytes": read, "flops": 4 * B * V}
    H, Hkv, D, T = (case[n] for n in ("H", "Hkv", "D", "T"))
    pairs = used = 0
    for n in lens:
        if case["op"] == "prefix":
            pairs += T * case["P"] + T * n + T * (T + 1) // 2
            used += n + T
        else:
            W, S = case["window"], case["sinks"]
            pairs += _seen_by(n + T, W, S) - _seen_by(n, W, S)
            far = max(0, n - W + 1)                                     # the first row in the first query's window
            used += n + T - far + min(S, far)
    used += case.get("P", 0)
    return {"bytes": w * (2 * B * H * T * D + 2 * Hkv * D * used), "flops": 4 * H * D * pairs}


def _seen_by(n, W, S):
    """Rows that the queries at positions 0 .. n - 1 see, all together."""
    near = n * (n + 1) // 2 if n <= W else W * (W + 1) // 2 + (n - W) * W
    m = n - W                                                           # queries p >= W: min(S, p - W + 1) sinks outside the window
    return near + (0 if m <= 0 else m * (m + 1) // 2 if m <= S else S * (S + 1) // 2 + (m - S) * S)


# ---------------------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "penalties":
        return _exact_penalties(s)
    B, H, Hkv, D, T = (case[n] for n in ("B", "H", "Hkv", "D", "T"))
    out = torch.zeros(B, T, H, D, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        for t0 in range(0, T, 1024):
            t1 = min(T, t0 + 1024)
            p = torch.arange(n + t0, n + t1, device="cuda")[:, None]
            if case["op"] == "prefix":
                cols = torch.arange(n + t1, device="cuda")
                ok = torch.cat([torch.ones(t1 - t0, case["P"], dtype=torch.bool, device="cuda"), cols[None] <= p], 1)
            else:
                start = max(0, n + t0 - case["window"] + 1)
                cols = torch.cat([torch.arange(min(case["sinks"], start), device="cuda"), torch.arange(start, n + t1, device="cuda")])
                ok = (cols[None] <= p) & ((cols[None] < case["sinks"]) | (p - cols[None] < case["window"]))
            for kh in range(Hkv):
                k, v = s["k"][b, kh, cols].double(), s["v"][b, kh, cols].double()
                if case["op"] == "prefix":
                    k, v = torch.cat([s["kp"][0, kh].double(), k]), torch.cat([s["vp"][0, kh].double(), v])
                for h in range(kh * (H // Hkv), (kh + 1) * (H // Hkv)):
                    z = (s["q"][b, h, t0:t1].double() @ k.T) * s["scaling"]
                    z[~ok] = -math.inf
                    out[b, t0:t1, h] = torch.softmax(z, -1) @ v
    return out.view(B, T, H * D)


def _exact_penalties(s):
    x = s["logits"].double()
    B, V = x.shape
    for b in range(B):
        n, n0 = int(s["n_tokens"][b]), int(s["n_prompt"][b])
        ids = s["tokens"][b, :n]
        seen = torch.unique(ids)
        r = s["repetition"][b].double()
        row = x[b]
        z = row[seen]
        row[seen] = torch.where(z > 0, z / r, z * r)
        used, count = torch.unique(ids[n0:], return_counts=True)
        row[used] -= s["frequency"][b].double() * count + s["presence"][b].double()
    if s["bias"] is not None:
        x += s["bias"].double()
    if s["allowed"] is not None:
        words = s["allowed"].long().bitwise_and(0xffffffff)
        bits = torch.stack([words >> i & 1 for i in range(32)], -1).flatten(1)[:, :V]
        x[(bits == 0).expand(B, V)] = -math.inf
    return x
