"""The windowed attention and the penalties as the models and the benchmark call them: a Mistral model whose cache slabs outgrow its
sliding window in static decode, its prefill through the windowed kernel, and e2e's greedy decode with penalties."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def build(monkeypatch, slab, window, extra=()):
    from baselines.monkeypatch import replace_mistral, set_model
    from benchmark import prefill
    monkeypatch.setenv("FASTKV_SLAB_CACHE", slab)
    a = prefill.parse_args(["--model_path", "mistral-7b", "--num_layers", "2", "--device", "cuda", "--method", "fastkv", "--max_capacity_prompts", "128",
                            "--tsp_len", "256", "--tsp_idx", "0", "--sliding_window", str(window), *extra])
    a.save_txt = False
    a.context_lengths = [600]
    replace_mistral("fastkv")
    torch.manual_seed(3)
    model = prefill.build_model(a, "cuda")
    set_model(model, a)
    return model, a


IDS = torch.randint(0, 1000, (1, 600), generator=torch.Generator().manual_seed(5))


def no_timer(fn):
    fn()
    torch.cuda.synchronize()
    return 0.0, None


def test_static_decode_keeps_to_the_sliding_window(monkeypatch):
    """128 rows per layer, a window of 48: the captured step over the slabs against attention in fp32 over the last 48 rows, layer by layer."""
    from benchmark import e2e
    from fastkv_amd import ops
    model, _ = build(monkeypatch, "1", 48)
    seen = []
    real = ops.decode_window_attention

    def spy(q, k, v, n, scaling, window=None, **kw):
        out = real(q, k, v, n, scaling, window=window, **kw)
        if not torch.cuda.is_current_stream_capturing():
            L = int(n.item())                                       # (after the call: rows 0 .. L - 1)
            lo = max(0, L - window)
            kk, vv = (t[:, :, lo:L].float().repeat_interleave(q.shape[1] // t.shape[1], 1) for t in (k, v))
            p = torch.softmax((q.float() @ kk.transpose(-1, -2).contiguous()) * scaling, -1)
            want = (p @ vv).transpose(1, 2).reshape(out.shape)
            seen.append((L, window, float((out.float() - want).abs().max()), float(want.abs().max())))
        return out

    monkeypatch.setattr(ops, "decode_window_attention", spy)
    ids = IDS.cuda()
    with torch.no_grad():
        out = model(ids, attention_mask=torch.ones_like(ids))
        pkv = out.past_key_values
        first = out.logits[:, -1].argmax(-1, keepdim=True)
        _, toks = e2e.graph_decode(model, pkv, first, 6, no_timer)
        assert [x[:2] for x in seen] == [(129, 48), (129, 48)]      # the eager step, two layers
        for _, _, off, size in seen:
            assert off <= 2 ** -10 * size + 1e-4                    # two roundings to fp16 of half a step each, and fp32 sums
        assert len(toks) == 6 and pkv.get_seq_length() == 134
        # the replayed steps: the same tokens as six eager static steps of a fresh cache
        out = model(ids, attention_mask=torch.ones_like(ids))
        pkv = out.past_key_values
        pkv.enable_static_decode(8)
        tok, again = first, []
        pos = torch.full((1, 1), pkv.get_seq_length(), dtype=torch.int64, device="cuda")
        for _ in range(6):
            o = model(input_ids=tok, past_key_values=pkv, position_ids=pos)
            tok = o.logits[:, -1].argmax(-1, keepdim=True)
            pos = pos + 1
            again.append(int(tok))
        assert again == toks


def test_a_window_as_long_as_the_slab_decodes_as_before(monkeypatch):
    from fastkv_amd import ops
    model, _ = build(monkeypatch, "1", 4096)
    monkeypatch.setattr(ops, "decode_window_attention", None)       # must not be called
    from benchmark import e2e
    ids = IDS.cuda()
    with torch.no_grad():
        out = model(ids, attention_mask=torch.ones_like(ids))
        _, toks = e2e.graph_decode(model, out.past_key_values, out.logits[:, -1].argmax(-1, keepdim=True), 4, no_timer)
    assert len(toks) == 4


def test_prefill_through_the_windowed_kernel(monkeypatch):
    """FASTKV_WINDOW_ATTENTION=1 against SDPA with the dense mask: logits of a two-layer fp16 model with a window of 100."""
    from fastkv_amd import ops
    model, _ = build(monkeypatch, "0", 100)
    ids = IDS.cuda()
    calls = []
    real = ops.window_attention
    monkeypatch.setattr(ops, "window_attention", lambda *a, **k: calls.append(k["window"]) or real(*a, **k))
    with torch.no_grad():
        want = model(ids, attention_mask=torch.ones_like(ids)).logits.float()
        assert not calls
        monkeypatch.setenv("FASTKV_WINDOW_ATTENTION", "1")
        got = model(ids, attention_mask=torch.ones_like(ids)).logits.float()
    assert calls == [100, 100]
    assert float((got - want).abs().max()) <= 2e-2 * float(want.abs().max())          # as the decode paths are compared


@pytest.mark.parametrize("slab", ["0", "1"])
def test_e2e_with_penalties(monkeypatch, slab):
    """Greedy decode with penalties: the benchmark's loops (eager, captured) pick what the formula picks from the step's own logits."""
    from benchmark import e2e
    model, args = build(monkeypatch, slab, 0, ("--repetition_penalty", "1.7", "--frequency_penalty", "0.4", "--presence_penalty", "0.2", "--genlen", "6",
                                               "--num_warmups", "0", "--random_tokens"))
    args.context_length = 600
    picked = []
    real = e2e.Penalties.apply

    def spy(self, logits):
        out = real(self, logits)
        if not torch.cuda.is_current_stream_capturing():
            x, n, n0 = logits[0, -1].double().cpu(), int(self.n[0]), int(self.n_prompt[0])
            said = self.tokens[0, :n].tolist()
            for v in set(said):
                x[v] = x[v] / float(torch.tensor(1.7)) if x[v] > 0 else x[v] * float(torch.tensor(1.7))
                c = said[n0:].count(v)
                x[v] -= float(torch.tensor(0.4)) * c + (float(torch.tensor(0.2)) if c else 0.0)
            # an fp32 chain of a few operations and one rounding to fp16
            assert float((out[0].double().cpu() - x).abs().max()) <= 2.0 ** -11 * float(x.abs().max()) + 1e-5
            picked.append(n)
        return out

    monkeypatch.setattr(e2e.Penalties, "apply", spy)
    res = e2e.main(model, args)
    assert res["genlen"] == 6
    # eager: prefill's choice and five steps; captured: prefill's choice, the eager first step (then replays)
    assert picked == ([600, 601, 602, 603, 604, 605] if slab == "0" else [600, 601])
