"""Beam search over the step engines: the search itself on a model that is a table, then the models' engines."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from onebit_amd.engine import MixedStep
    from onebit_amd.llama import KVCache, OneBitLlamaConfig, build_synthetic_model
    from onebit_amd.search import HybridBeams, LlamaBeams, beam_search

F64 = torch.float64


def reference(logits_of, prompt, beams, n_new, eos=frozenset(), penalty=1.0, early=False, keep=None):
    """Beam search over all beams x vocab continuations, in 64 bits.  ``logits_of(tokens)`` -> [vocab]."""
    keep = keep or (1 + max(1, len(eos))) * beams
    live, done = [(0.0, ())], []

    def finish(score, toks):
        done.append((score / len(toks) ** penalty, toks))
        done.sort(key=lambda d: -d[0])
        del done[beams:]
    stopped = False
    for _ in range(n_new):
        every = []
        for b, (score, toks) in enumerate(live):
            lp = torch.log_softmax(logits_of(prompt + list(toks)).double(), -1)
            every += [(-(score + v), b, t) for t, v in enumerate(lp.tolist()) if v > -math.inf]
        every.sort()
        nxt = []
        for rank, (s, b, t) in enumerate(every[:keep]):
            if t in eos:
                if rank < beams and len(nxt) < beams:
                    finish(-s, live[b][1] + (t,))
            elif len(nxt) < beams:
                nxt.append((-s, live[b][1] + (t,)))
        live = nxt
        if not live or (len(done) == beams and (early or live[0][0] / len(live[0][1]) ** penalty <= done[-1][0])):
            stopped = True
            break
    if not stopped:
        for s, toks in live:
            finish(s, toks)
    return done


class Table:
    """An engine whose logits are a random function of the last two tokens and the position (without it, two paths that take the same transitions in another
    order have equal scores, and roundings decide); it keeps every slot's tokens and checks that each step finds in a slot what its hypothesis has seen so far."""

    def __init__(self, batch, beams, vocab, seed, scale=2.0, dtype=torch.float32):
        g = torch.Generator().manual_seed(seed)
        self.table = (scale * torch.randn(vocab, vocab, generator=g)).to(dtype)
        self.shift = torch.randn(vocab, generator=g)
        self.place = torch.randn(64, vocab, generator=g)
        self.batch, self.beams, self.vocab, self.max_len, self.device, self.dtype = batch, beams, vocab, 1000, torch.device("cuda"), dtype
        self.held, self.moves = {}, 0

    def of(self, tokens):
        return (self.table[tokens[-1]].float() + self.place[len(tokens)] + (self.shift[tokens[-2]] * self.shift if len(tokens) > 1 else 0)).to(self.dtype)

    def prime(self, prompts):
        self.prompts = [list(p) for p in prompts]
        return torch.stack([self.of(p) for p in prompts]).cuda()

    def spread(self, lengths):
        self.held = {(i, s): [] for i in range(self.batch) for s in range(self.beams)}

    def advance(self, live, slots, tokens, positions, lengths):
        rows = []
        for i in live:
            assert sorted(slots[i]) == list(range(self.beams))
            for s, t in zip(slots[i], tokens[i]):
                self.held[i, s] = self.held[i, s] + [t]
                assert positions[i] == lengths[i] + len(self.held[i, s]) - 1
                rows.append(self.of(self.prompts[i] + self.held[i, s]))
        return torch.stack(rows).cuda()

    def move(self, parents, first, end):
        self.moves += 1
        p = parents.cpu().tolist()
        self.held = {(i, s): list(self.held[i, p[i][s]]) for i, s in self.held}


@pytest.mark.parametrize("batch, beams, vocab, n_new, eos, penalty, early", [
    (1, 1, 40, 6, (), 1.0, False), (1, 4, 40, 12, (), 1.0, False), (3, 5, 97, 20, (), 1.0, False), (4, 4, 31, 25, (3,), 1.0, False), (4, 4, 31, 25, (3,), 1.0, True),
    (2, 3, 29, 30, (3, 7), 0.6, False), (2, 8, 500, 9, (5,), 2.0, False), (1, 32, 200, 6, (), 1.0, False), (2, 6, 4, 8, (), 1.0, False), (2, 3, 2, 7, (1,), 1.0, False)])
def test_search_on_a_table(batch, beams, vocab, n_new, eos, penalty, early):
    eng = Table(batch, beams, vocab, seed=beams + vocab)
    prompts = [[(7 * i + 3) % vocab] * (1 + i) for i in range(batch)]
    got = beam_search(eng, prompts, n_new, set(eos) or None, penalty, early)
    for p, hyps in zip(prompts, got):
        want = reference(eng.of, p, beams, n_new, frozenset(eos), penalty, early, keep=min(64, (1 + max(1, len(eos))) * beams))
        assert [t for _, t in hyps] == [list(t) for _, t in want]
        # (scores pass through fp32 at every step, and are off by 2^-24 of themselves and of a few units each time)
        assert all(abs(a - b) <= n_new * 2.0 ** -23 * (1 + abs(b) * n_new) for (a, _), (b, _) in zip(hyps, want))
    assert eng.moves > 0 or beams == 1 or vocab - len(eos) == 1          # (one token that does not end: one path)


@pytest.mark.parametrize("default", [torch.float64, torch.float16])
def test_search_under_another_default_type(default):
    """Scores are float32 whatever type new tensors have."""
    eng = Table(2, 3, 41, seed=5)
    want = beam_search(eng, [[1], [2, 3]], 6)
    torch.set_default_dtype(default)
    try:
        assert beam_search(eng, [[1], [2, 3]], 6) == want
    finally:
        torch.set_default_dtype(torch.float32)


def test_one_copy_to_the_host_a_step(monkeypatch):
    copies = []
    for name in ("tolist", "cpu", "item"):
        def count(self, *args, _plain=getattr(torch.Tensor, name), **kw):
            copies.append(self.is_cuda)
            return _plain(self, *args, **kw)
        monkeypatch.setattr(torch.Tensor, name, count)
    beam_search(Table(3, 1, 41, seed=5), [[1], [2], [3]], 7)          # (one hypothesis each: nothing moves)
    assert sum(copies) == 7


class Script(Table):
    """Logits as given, by step and row."""

    def __init__(self, batch, beams, steps):
        super().__init__(batch, beams, len(steps[0][0]), seed=1)
        self.steps = [torch.tensor(s).cuda() for s in steps]

    def prime(self, prompts):
        return self.steps.pop(0)

    def advance(self, live, slots, tokens, positions, lengths):
        return self.steps.pop(0)


def test_a_prompt_that_has_ended_moves_nothing():
    """In the second step the first prompt's two hypotheses end and its better one would go on twice; the second prompt's go on where they are."""
    low = -30.0
    first = [[low, 1.0, 0.0, low, low], [low, 1.0, 0.0, low, low]]
    both = [[5.0, low, 0.0, -0.1, low], [5.0, low, -9.0, low, low], [low, low, 5.0, low, low], [low, low, low, 5.0, low]]
    last = [[low, low, 5.0, low, low], [low, low, low, 5.0, low]]
    eng = Script(2, 2, [first, both, last])
    found = beam_search(eng, [[1], [2]], 3, eos={0}, early_stopping=True)
    assert [t for _, t in found[0]] == [[1, 0], [2, 0]] and [t for _, t in found[1]] == [[1, 2, 2], [2, 3, 3]]
    assert eng.moves == 0


def test_search_refusals():
    eng = Table(2, 3, 11, seed=1)
    for prompts, n in (([[1]], 4), ([[1], []], 4), ([[1], [2]], 1000)):
        with pytest.raises(ValueError):
            beam_search(eng, prompts, n)


# ----------------------------------------------------------------------------------------------------------------- 1-bit LLaMA --
def _llama(**kw):
    cfg = dict(vocab_size=96, hidden_size=256, intermediate_size=352, num_hidden_layers=2, num_attention_heads=4, max_position_embeddings=1024)
    return build_synthetic_model(OneBitLlamaConfig(**{**cfg, **kw}), seed=1, device="cuda")


@pytest.mark.parametrize("kv_heads", [4, 1])
@pytest.mark.parametrize("length", [1, 40, 700])
def test_step_with_a_shared_prefix(kv_heads, length):
    """Rows that share a prompt's slot give the logits of rows that each hold a copy of it."""
    model = _llama(num_key_value_heads=kv_heads)
    g = torch.Generator().manual_seed(length)
    prompts = [torch.randint(0, 96, (n,), generator=g).tolist() for n in (length, 30)]
    tails = [[torch.randint(0, 96, (5,), generator=g).tolist() for _ in range(n)] for n in (3, 2)]
    cache = KVCache(model.config, 12, 1000, "cuda", torch.float16)
    step = MixedStep(model, cache.layers, 12, 1000, keep_logits=True)
    step.launch([(5, 0, prompts[0]), (6, 0, prompts[1])])
    flat = [(s, len(p), t) for p, s0, ts in zip(prompts, (0, 3), tails) for s, t in enumerate(ts, s0)]
    for k in range(5):
        step.launch([(s, n + k, [t[k]]) for s, n, t in flat], prefixes=[(3, 5, len(prompts[0])), (2, 6, len(prompts[1]))])
    shared = step.logits[:5].clone()
    step.launch([(s, 0, p) for p, s0, ts in zip(prompts, (0, 3), tails) for s in range(s0, s0 + len(ts))])
    for k in range(5):
        step.launch([(s, n + k, [t[k]]) for s, n, t in flat])
    own = step.logits[:5]
    # both round activations to fp16 (2^-11) some twenty times on the way and differ in the scores' and weights' rounding
    assert float((shared.float() - own.float()).norm() / own.float().norm()) < 20 * 2.0 ** -11
    for bad in ([(4, 5, length)], [(3, 5, length)], [(3, 5, length), (2, 12, 30)], [(3, 5, length), (2, 6, 1001)], [(3, 5, length + 6), (2, 6, 30)], [(6, 5, length)]):
        with pytest.raises(ValueError):
            step.launch([(s, n + 4, [t[4]]) for s, n, t in flat], prefixes=bad)


def _log_prob(model, prompt, tokens):
    lg = model(torch.tensor([prompt + tokens[:-1]], device="cuda"))[0].double()
    lp = torch.log_softmax(lg, -1)
    return sum(lp[len(prompt) - 1 + i, t].item() for i, t in enumerate(tokens)), lg.abs().max().item()


@pytest.mark.parametrize("beams, prompts, eos", [(4, [(9, 9)], None), (3, [(200, 1), (5, 2), (64, 3)], None), (5, [(1, 4), (33, 5)], {7, 8}), (32, [(12, 6)], None)])
def test_llama_hypotheses_have_their_scores(beams, prompts, eos):
    model = _llama()
    prompts = [torch.randint(0, 96, (n,), generator=torch.Generator().manual_seed(s)).tolist() for n, s in prompts]
    eng = LlamaBeams(model, len(prompts), beams, 256)
    for _ in range(2):                                               # (the second search finds the slots as the first left them)
        found = beam_search(eng, prompts, 12, eos)
    for p, hyps in zip(prompts, found):
        assert len(hyps) == beams and len({tuple(t) for _, t in hyps}) == beams
        assert [s for s, _ in hyps] == sorted((s for s, _ in hyps), reverse=True)
        greedy, tol = None, None
        for score, toks in hyps[:4]:
            lp, size = _log_prob(model, p, toks)
            # a logit is off by some twenty roundings to fp16 of values of the logits' size, on both sides of the subtraction
            tol = 2 * 20 * 2.0 ** -11 * size
            assert abs(score - lp / len(toks)) <= tol, (score, lp / len(toks))
        if eos is None:
            row = model.generate(torch.tensor([p], device="cuda"), 12)[0, len(p):].tolist()
            greedy = _log_prob(model, p, row)[0] / 12
            assert hyps[0][0] >= greedy - 2 * tol or beams < 4


def test_llama_generate_native():
    model = _llama()
    ids = torch.randint(0, 96, (2, 20), generator=torch.Generator().manual_seed(3)).cuda()
    out = model.generate_native(ids, 10, num_beams=4)
    assert out.shape == (2, 30) and torch.equal(out[:, :20], ids)
    assert torch.equal(out, model.generate_native(ids, 10, num_beams=4))
    assert torch.equal(model.generate_native(ids, 10, num_beams=1), model.generate_native(ids, 10))
    eos = int(out[0, 22])
    cut = model.generate_native(ids, 10, eos_token_id=eos, pad_token_id=95, num_beams=4, early_stopping=True)
    assert cut.shape[0] == 2 and cut.shape[1] <= 30
    for bad in (0, 33, -1):
        with pytest.raises(ValueError):
            model.generate_native(ids, 10, num_beams=bad)
    with pytest.raises(ValueError):
        model.generate_native(ids, 1010, num_beams=2)


# -------------------------------------------------------------------------------------------------------------- hybrid decoders --
def _lebepel(dtype):
    from onebit_amd.lebepel import LebepelConfig, build_synthetic_model as build
    mlp = {"kind": "dense", "ff": 72}
    cfg = LebepelConfig(vocab_size=96, width=80, norm_eps=1e-5, residual_mult=0.5, logit_softcap=20.0, max_positions=128, loop={"start": 0, "stop": 2, "times": 2},
                        layers=[{"type": "mamba2", "mixer": dict(heads=4, groups=2, state=16, vdim=24, conv=4, norm_groups=2), "mlp": mlp},
                                {"type": "attention", "mixer": dict(heads=4, kv_heads=2, dim=24, vdim=32, scale=0.2), "mlp": mlp}])
    return build(cfg, seed=3, device="cuda", dtype=dtype)


def _serotar(dtype):
    from onebit_amd.serotar import SerotarConfig, build_synthetic_model as build
    mix = dict(heads=3, dim=24, vdim=40, q_rank=36, kv_rank=72, scale=0.2)
    moe = {"kind": "moe", "expert": {"ff": 40}, "shared": {"ff": 56}, "router": {"experts": 6, "identity": 2, "top": 2, "groups": {"count": 4, "keep": 2}}}
    cfg = SerotarConfig(vocab_size=96, width=72, norm_eps=1e-5, embed_scale=2.0, bigram={"buckets": 53, "mul_prev": 5, "mul_cur": 3}, side_dim=12,
                        layers=[{"type": "latent_attention", "mixer": mix, "mlp": {"kind": "dense", "ff": 88}}, {"type": "latent_attention", "mixer": mix, "mlp": moe}])
    return build(cfg, seed=3, device="cuda", dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("make", [_lebepel, _serotar])
def test_hybrid_search(make, dtype):
    """Every hypothesis's score is that of its tokens through a whole forward pass: keys, latent rows, recurrent states, convolution rings and token histories
    have followed it from slot to slot.  In fp32 the hypotheses are the reference search's."""
    model = make(dtype)
    prompts = [torch.randint(0, 96, (n,), generator=torch.Generator().manual_seed(n)).tolist() for n in (37, 9)]
    eng = HybridBeams(model, 2, 4, 80)
    for _ in range(2):
        found = beam_search(eng, prompts, 20)
    for p, hyps in zip(prompts, found):
        if dtype == torch.float32:
            want = reference(lambda t: model.forward(torch.tensor([t], device="cuda"))[0, -1].cpu(), p, 4, 20)
            assert [t for _, t in hyps] == [list(t) for _, t in want]
        for score, toks in hyps:
            lp, size = _log_prob(model.forward, p, toks)
            tol = 2 * 20 * size * (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -18)
            assert abs(score - lp / len(toks)) <= tol, (score, lp / len(toks))


def test_hybrid_generate():
    model = _lebepel(torch.bfloat16)
    ids = torch.randint(0, 96, (3, 11), generator=torch.Generator().manual_seed(3)).cuda()
    out = model.generate(ids, 8, num_beams=3)
    assert out.shape == (3, 19) and torch.equal(out[:, :11], ids)
    assert torch.equal(out, model.generate_native(ids, 8, num_beams=3))


def test_command_line(tmp_path, capsys):
    from onebit_amd.checkpoint import write_safetensors
    from onebit_amd.cli import main
    from onebit_amd.lebepel import LebepelConfig, synthetic_weights
    from onebit_amd.registry import load_model
    import json
    raw = {"architecture": "Lebepel", "vocab": 50, "width": 64, "norm": {"eps": 1e-5}, "residual_mult": 0.5, "logit_softcap": 20.0, "max_positions": 128,
           "layers": [{"type": "mamba2", "mixer": dict(heads=4, groups=2, state=16, vdim=24, conv=4, norm_groups=2), "mlp": {"kind": "dense", "ff": 72}},
                      {"type": "attention", "mixer": dict(heads=4, kv_heads=2, dim=24, vdim=32, scale=0.2), "mlp": {"kind": "dense", "ff": 72}}]}
    (tmp_path / "config.json").write_text(json.dumps(raw))
    write_safetensors(str(tmp_path / "model.safetensors"), synthetic_weights(LebepelConfig.from_dict(raw), 6))
    prompts = [[3, 4, 9, 30, 7], [8]]
    run = lambda *extra: main(["generate", "--model", str(tmp_path), "--dtype", "float32", "--max-new-tokens", "5", *extra] + [x for p in prompts for x in ("--prompt", ",".join(map(str, p)))])
    assert run("--num-beams", "3") == 0
    rows = [json.loads(l)["tokens"] for l in capsys.readouterr().out.splitlines() if l.startswith("{")]
    model = load_model(str(tmp_path), dtype=torch.float32)
    for p, row in zip(prompts, rows):
        assert row == list(reference(lambda t: model.forward(torch.tensor([t], device="cuda"))[0, -1].cpu(), p, 3, 5)[0][1])
    end = rows[0][1]
    assert run("--num-beams", "2", "--eos", str(end), "--length-penalty", "0.5") == 0
    ended = [json.loads(l)["tokens"] for l in capsys.readouterr().out.splitlines() if l.startswith("{")]
    for p, row in zip(prompts, ended):
        assert row == list(reference(lambda t: model.forward(torch.tensor([t], device="cuda"))[0, -1].cpu(), p, 2, 5, frozenset([end]), 0.5)[0][1])


def test_shared_rows_next_to_prompts():
    """A step that carries prompt chunks beside rows that share a prefix gives each what it gives alone."""
    model = _llama()
    g = torch.Generator().manual_seed(4)
    tok = lambda n: torch.randint(0, 96, (n,), generator=g).tolist()
    base, other, chunk = tok(300), tok(70), tok(40)
    cache = KVCache(model.config, 8, 400, "cuda", torch.float16)
    step = MixedStep(model, cache.layers, 8, 400, keep_logits=True)
    step.launch([(6, 0, base), (5, 0, other)])
    step.launch([(0, 300, [1]), (7, 0, chunk), (1, 300, [2]), (2, 70, [3])], prefixes=[(2, 6, 300), (1, 5, 70)])
    got = step.logits[:4].clone()
    for i, seq in enumerate((base + [1], chunk, base + [2], other + [3])):
        step.launch([(3, 0, seq)])
        want = step.logits[0]
        assert float((got[i].float() - want.float()).norm() / want.float().norm()) < 20 * 2.0 ** -11
