"""Beam search over the native step engines: per prompt, the ``beams`` continuations with the largest sums of log probabilities are followed,
all prompts' hypotheses in one step.

The 1-bit LLaMA's hypotheses share their prompt's keys and values: they lie in one slot of their own, and the decode attention reads them once
for all hypotheses (``shared_prefix_attention`` inside ``onebit_mixed_step_shared``).  The hybrid decoders' hypotheses start from copies of their
prompt's state.  A step's candidates come from ``beam_select``; a hypothesis that goes on keeps its slot, and only where one goes on more than
once its states are copied, to the slot of one that has ended (``reorder_slots``)."""
from __future__ import annotations

import math
from typing import Dict, List, Optional, Sequence, Set, Tuple

import torch

from .beam import MAX_BEAMS, MAX_KEEP, beam_select_workspace, reorder_slots, select_packed

_PRIME_ROWS = 8192          # prompt tokens of one step, unless a single prompt has more


def _prime(step, first_slot: int, stride: int, prompts: Sequence[Sequence[int]]) -> torch.Tensor:
    """The prompts into slots first_slot, first_slot + stride, ..; the logits behind their last tokens."""
    rows, items = [], []

    def flush():
        step.launch([(s, 0, p) for s, p in items])
        rows.append(step.logits[:len(items)].clone())
        items.clear()
    for i, p in enumerate(prompts):
        if items and sum(len(q) for _, q in items) + len(p) > _PRIME_ROWS:
            flush()
        items.append((first_slot + i * stride, list(p)))
    flush()
    return torch.cat(rows) if len(rows) > 1 else rows[0]


class LlamaBeams:
    """Slots of a 1-bit LLaMA: hypothesis b of prompt i in slot i beams + b, the prompt itself in slot batch beams + i.  Every slot is max_len long, since a token's place
    in its slot is its position: batch (beams + 1) of them."""

    def __init__(self, model, batch: int, beams: int, max_len: int):
        from .engine import MixedStep
        from .llama import KVCache
        self.batch, self.beams, self.max_len = batch, beams, max_len
        n = batch * (beams + 1)
        self.caches = KVCache(model.config, n, max_len, model.lm_head.weight.device, torch.float16).layers
        chunk = max(256, -(-max_len // (64 * 64)) * 64)
        self.step = MixedStep(model, self.caches, n, max_len, max_rows=64, attn_chunk=chunk, keep_logits=True)
        self.device, self.vocab = self.step.dev, model.config.vocab_size

    def prime(self, prompts):
        return _prime(self.step, self.batch * self.beams, 1, prompts)

    def spread(self, lengths):
        pass

    def advance(self, live, slots, tokens, positions, lengths):
        items = [(i * self.beams + s, positions[i], [t]) for i in live for s, t in zip(slots[i], tokens[i])]
        self.step.launch(items, prefixes=[(self.beams, self.batch * self.beams + i, lengths[i]) for i in live])
        return self.step.logits[:len(items)]

    def move(self, parents, first: int, end: int):
        reorder_slots([t for kv in self.caches for t in kv], parents, first=first, count=end - first)


class HybridBeams:
    """Slots of a hybrid decoder: hypothesis b of prompt i in slot i beams + b, started from a copy of the prompt's state in slot i beams."""

    def __init__(self, model, batch: int, beams: int, max_len: int):
        self.batch, self.beams, self.max_len = batch, beams, max_len
        self.step = model.step_engine(batch * beams, max_len)
        self.device, self.vocab = self.step.dev, model.vocab_size

    def prime(self, prompts):
        return _prime(self.step, 0, self.beams, prompts)

    def spread(self, lengths):
        self.move(torch.zeros(self.batch, self.beams, dtype=torch.int32, device=self.device), 0, max(lengths))

    def advance(self, live, slots, tokens, positions, lengths):
        items = [(i * self.beams + s, positions[i], [t]) for i in live for s, t in zip(slots[i], tokens[i])]
        self.step.launch(items)
        return self.step.logits[:len(items)]

    def move(self, parents, first: int, end: int):
        st = self.step.states
        whole = [t for (i, _), run in zip(st.decoder.runs, st.runs) if st.decoder.packed[i].c.kind == 1 for t in run]
        rows = [t for (i, _), run in zip(st.decoder.runs, st.runs) if st.decoder.packed[i].c.kind == 0 for t in run]
        tiles = [t.view(t.shape[0], 1, t.shape[1], -1) for (i, _), run in zip(st.decoder.runs, st.runs) if st.decoder.packed[i].c.kind == 2 for t in run]
        if st.tokens is not None:
            rows.append(st.tokens.view(st.n_slots, 1, st.max_len, 1))
        reorder_slots(whole, parents)
        reorder_slots(rows, parents, first=first, count=end - first)
        reorder_slots(tiles, parents, first=first // 16, count=-(-end // 16) - first // 16)


class _Prompt:
    """One prompt's search: its hypotheses (score, tokens, slot), best first, and the finished ones (length-normalised score, tokens)."""

    def __init__(self, beams: int, length_penalty: float, early_stopping: bool):
        self.beams, self.penalty, self.early = beams, length_penalty, early_stopping
        self.live: List[Tuple[float, List[int], int]] = [(0.0, [], 0)]
        self.finished: List[Tuple[float, List[int]]] = []
        self.done = False

    def _finish(self, score: float, tokens: List[int]):
        self.finished.append((score / len(tokens) ** self.penalty, tokens))
        self.finished.sort(key=lambda f: -f[0])                          # (stable: the earlier one of equals stays in front)
        del self.finished[self.beams:]

    def take(self, candidates, eos: Optional[Set[int]]) -> List[int]:
        """The next hypotheses from the step's candidates (score, beam, token), best first; the parent slot of every slot."""
        nxt = []
        for rank, (score, beam, token) in enumerate(candidates):
            if beam < 0 or len(nxt) == self.beams:
                break
            tokens = self.live[beam][1] + [token]
            if eos is not None and token in eos:
                if rank < self.beams:                                    # (worse than all that could go on: not a result)
                    self._finish(score, tokens)
            else:
                nxt.append((score, tokens, beam))
        free = sorted(set(range(self.beams)) - {self.live[b][2] for _, _, b in nxt})
        taken, parents, live = set(), list(range(self.beams)), []
        for score, tokens, beam in nxt:
            slot = source = self.live[beam][2]
            if source in taken:
                slot = free.pop(0)
                parents[slot] = source
            taken.add(slot)
            live.append((score, tokens, slot))
        self.live = live
        if not live:
            self.done = True
        elif len(self.finished) == self.beams:
            # the best that a live hypothesis could still become if it lost nothing more, at its present length
            self.done = self.early or live[0][0] / len(live[0][1]) ** self.penalty <= self.finished[-1][0]
        return parents

    def results(self) -> List[Tuple[float, List[int]]]:
        if not self.done:
            for score, tokens, _ in self.live:
                self._finish(score, tokens)
        return self.finished


def _candidates(beams: int, eos: Optional[Set[int]]) -> int:
    keep = (1 + max(1, len(eos or ()))) * beams
    if keep > MAX_KEEP:
        raise ValueError(f"beam_search: {beams} beams with {len(eos or ())} end tokens look at {keep} candidates a step, at most {MAX_KEEP} are kept")
    return keep


@torch.no_grad()
def beam_search(engine, prompts: Sequence[Sequence[int]], max_new_tokens: int, eos: Optional[Set[int]] = None, length_penalty: float = 1.0,
                early_stopping: bool = False) -> List[List[Tuple[float, List[int]]]]:
    """Per prompt the finished hypotheses, best first, as (score, tokens): the sum of the new tokens' log probabilities over their number to the power
    ``length_penalty``, an end token counted.  A prompt ends when it has ``beams`` finished hypotheses and (``early_stopping`` or) no live one that would
    beat the worst of them as it stands, or after ``max_new_tokens``, where the live ones count as finished.  A step looks at beams x (1 + end tokens) candidates, so
    that ``beams`` go on however many of them end; 64 at most."""
    B, W = len(prompts), engine.beams
    if B != engine.batch or any(len(p) < 1 for p in prompts):
        raise ValueError(f"beam_search: {B} prompts of at least one token for an engine of {engine.batch}")
    if max(len(p) for p in prompts) + max_new_tokens > engine.max_len:
        raise ValueError("beam_search: prompt + max_new_tokens exceeds the engine's slots")
    lengths = [len(p) for p in prompts]
    keep = _candidates(W, eos)
    if max_new_tokens < 1:
        return [[(0.0, [])] for _ in prompts]
    workspace = beam_select_workspace(B * W, engine.vocab, keep, engine.device)
    logits = engine.prime(prompts)
    engine.spread(lengths)
    states = [_Prompt(W, length_penalty, early_stopping) for _ in prompts]
    live, scores, per = list(range(B)), torch.zeros(B, dtype=torch.float32, device=engine.device), 1
    for step in range(max_new_tokens):
        found = select_packed(logits, scores, per, keep, workspace).cpu()
        v, b, t = found[0].view(torch.float32).tolist(), found[1].tolist(), found[2].tolist()
        moves, moved = [list(range(W)) for _ in range(B)], False
        for g, i in enumerate(live):
            parents = states[i].take(list(zip(v[g], b[g], t[g])), eos)
            if not states[i].done:                                       # (nobody reads an ended prompt's slots again)
                moves[i] = parents
                moved = moved or parents != list(range(W))
        live = [i for i in live if not states[i].done]
        if not live or step + 1 == max_new_tokens:
            break
        # (a prompt with fewer hypotheses than beams is filled up with dead ones, in the slots that are left)
        slots, tokens, flat = {}, {}, []
        for i in live:
            hyps = states[i].live
            spare = sorted(set(range(W)) - {h[2] for h in hyps})
            slots[i] = [h[2] for h in hyps] + spare
            tokens[i] = [h[1][-1] for h in hyps] + [0] * len(spare)
            flat += [h[0] for h in hyps] + [-math.inf] * len(spare)
        if moved and step:
            engine.move(torch.tensor(moves, dtype=torch.int32).to(engine.device), min(lengths[i] for i in live), max(lengths[i] for i in live) + step)
        scores, per = torch.tensor(flat, dtype=torch.float32).to(engine.device), W
        logits = engine.advance(live, slots, tokens, {i: lengths[i] + step for i in live}, lengths)
    return [s.results() for s in states]


def beam_rows(model, prompts: List[List[int]], max_new_tokens: int, max_positions: int, engines: Dict, beams: int, eos=None, length_penalty: float = 1.0,
              early_stopping: bool = False) -> List[List[int]]:
    """The best hypothesis of every prompt (its new tokens, an end token last if it ended), on slots that stay in ``engines`` until a search of other
    (prompts, beams, length bucket) needs its own."""
    if not 1 <= beams <= MAX_BEAMS:
        raise ValueError(f"num_beams must be in 1 .. {MAX_BEAMS}")
    _candidates(beams, eos)                                              # (what a search would refuse, before its slots take memory)
    if len(prompts) < 1 or any(len(p) < 1 for p in prompts):
        raise ValueError("beam search needs prompts of at least one token")
    longest = max(len(p) for p in prompts) + max_new_tokens
    if longest > max_positions:
        raise ValueError("prompt + max_new_tokens exceeds max_position_embeddings")
    key = ("beams", len(prompts), beams, min(-(-longest // 256) * 256, max_positions))
    eng = engines.get(key)
    if eng is None:
        for k in [k for k in engines if k[0] == "beams"]:                # (prompts x (beams + 1) slots of the whole length each: one search's at a time)
            del engines[k]
        if len(engines) >= 4:
            engines.clear()
        from .hybrid import HybridDecoder
        eng = engines[key] = (HybridBeams if isinstance(model, HybridDecoder) else LlamaBeams)(model, len(prompts), beams, key[3])
    found = beam_search(eng, prompts, max_new_tokens, eos, length_penalty, early_stopping)
    if not all(found):
        raise RuntimeError(f"beam search: no continuation of prompt {[bool(f) for f in found].index(False)} has a probability (NaN or infinite logits)")
    return [r[0][1] for r in found]


@torch.no_grad()
def generate_beams(model, input_ids: torch.Tensor, max_new_tokens: int, eos_token_id, pad_token_id, num_beams: int, length_penalty: float, early_stopping: bool,
                   engines: Dict) -> torch.Tensor:
    """``generate``'s contract for a hybrid decoder: the prompts [B, S] followed by their best hypotheses, padded to the longest."""
    from .serving import cut_at_eos, eos_set
    if input_ids.dim() != 2:
        raise ValueError("input_ids must be [B, S]")
    if max_new_tokens < 1:
        return input_ids
    eos, pad = eos_set(eos_token_id, pad_token_id, input_ids.shape[0])
    rows = beam_rows(model, input_ids.tolist(), max_new_tokens, model.max_positions, engines, num_beams, eos, length_penalty, early_stopping)
    return torch.cat([input_ids.to(model.device), torch.tensor(cut_at_eos(rows, eos, pad), dtype=input_ids.dtype, device=model.device)], dim=1)
