"""Beam search's operators, as a serving program calls them: what they are measured on, beside their plain forms.

  attention   single-token rows of several sequences that share a prefix of their keys and values: the prefix is stored once, each
              sequence's later positions in a cache slot of its own
  select      the next hypotheses of a beam search: the best continuations over beams and vocabulary, from logits and running scores
  reorder     the surviving hypotheses' states brought to the slots that go on with them, in place

Sizes: head counts and widths of LLaMA-7B / 13B and of the small models of the tests, and generic ones; a full batch has 64 rows."""
from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"
DTYPES = {"f16": torch.float16, "f32": torch.float32}

# (heads, key / value heads, head size)
HEADS = [(2, 2, 64), (8, 8, 64), (32, 32, 128), (40, 40, 128), (32, 8, 128), (64, 8, 128), (16, 2, 80), (12, 4, 96), (32, 1, 64), (5, 5, 40)]
VOCABS = [(512, 512), (32000, 32000), (50257, 50264), (128256, 128256), (999, 1003)]          # (tokens, row pitch of the logits)


def _attention(name, rows, groups, prefix, tail, heads, kv_heads, dim, ragged=False, idle=0):
    return {"name": name, "op": "attention", "rows": rows, "groups": groups, "prefix": prefix, "tail": tail, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "ragged": ragged, "idle": idle}


def _select(name, groups, beams, keep, vocab, pitch, dtype, banned=0, first=False):
    return {"name": name, "op": "select", "groups": groups, "beams": beams, "keep": keep, "vocab": vocab, "pitch": pitch, "dtype": dtype,
            "banned": banned, "first": first}


def _reorder(name, buffers, groups, beams, forks, outer, length, row, first, count, dtype):
    return {"name": name, "op": "reorder", "buffers": buffers, "groups": groups, "beams": beams, "forks": forks, "outer": outer, "length": length,
            "row": row, "first": first, "count": count, "dtype": dtype}


def listed():
    return [
        # four hypotheses of a small model a few tokens behind a short prompt: latency
        _attention("attention_small", 4, 1, 96, 9, 2, 2, 64),
        # one prompt of half the context, eight hypotheses, 7B heads
        _attention("attention_beams_7b", 8, 1, 1000, 48, 32, 32, 128),
        # a full server whose requests share a long instruction text; answers of many lengths, some slots idle
        _attention("attention_server_13b", 64, 1, 2040, 300, 40, 40, 128, ragged=True, idle=3),
        # eight prompts of odd lengths at once (one without any prefix), four hypotheses each, grouped heads
        _attention("attention_prompts_grouped", 32, 8, 5001, 130, 32, 8, 128, ragged=True),
        # a document that 64 requests ask about
        _attention("attention_document", 64, 1, 32768, 1024, 64, 8, 128, ragged=True),
        # four hypotheses over a small vocabulary: latency
        _select("select_small", 1, 4, 8, 512, 512, "f32"),
        # one search of eight hypotheses, LLaMA's vocabulary, logits as the step engine leaves them
        _select("select_beams_7b", 1, 8, 16, 32000, 32000, "f16"),
        # the first token of 16 prompts: one live row each
        _select("select_first", 16, 1, 8, 32000, 32000, "f32", first=True),
        # 64 searches of four, an odd vocabulary inside wider rows, some tokens banned
        _select("select_many", 64, 4, 8, 50257, 50264, "f16", banned=1000),
        # two small layers, four hypotheses
        _reorder("reorder_small", 4, 1, 4, 1, 2, 64, 64, 16, 9, "f16"),
        # 7B: 32 layers' keys and values behind a prompt of 150 tokens, four searches of four
        _reorder("reorder_7b", 64, 4, 4, 2, 32, 224, 128, 150, 64, "f16"),
        # recurrent states of a state-space model's layers, whole: 16 searches of four
        _reorder("reorder_states", 16, 16, 4, 1, 64, 64, 64, 0, 64, "f32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    most = {"attention": 3e11, "select": 1.2e8, "reorder": 7e8}            # operations / bytes of the largest listed case of a kind
    while True:
        op = rng.choice(["attention", "attention", "select", "reorder"])
        if op == "attention":
            h, hkv, d = rng.choice(HEADS)
            rows = rng.choice([1, 2, 3, 4, 8, 12, 17, 32, 48, 64])
            case = _attention("", rows, rng.randint(1, min(rows, 8)), _log_int(rng, 1, 32768), _log_int(rng, 1, 1024), h, hkv, d,
                              ragged=rng.random() < 0.7, idle=rng.choice([0, 0, rows // 8]))
            cost = work(case)["flops"]
            size = (case["rows"] * case["tail"] + case["groups"] * case["prefix"]) * hkv * d * 4
            if size > 4 << 30:
                continue
        elif op == "select":
            v, pitch = rng.choice(VOCABS)
            beams = rng.choice([1, 2, 3, 4, 5, 8, 16, 32])
            case = _select("", rng.choice([1, 2, 7, 16, 33, 64]), beams, min(2 * beams, 64), v, pitch, rng.choice(["f16", "f32"]),
                           banned=rng.choice([0, 0, 17, v // 3]), first=beams == 1)
            cost = work(case)["bytes"]
        else:
            beams = rng.choice([2, 3, 4, 8, 16])
            length = _log_int(rng, 16, 512)
            first = rng.randint(0, length - 1)
            case = _reorder("", rng.choice([2, 7, 16, 64]), rng.randint(1, 8), beams, rng.randint(1, beams - 1), rng.choice([1, 8, 32]), length,
                            rng.choice([40, 64, 128]), first, rng.randint(1, length - first), rng.choice(["f16", "f32"]))
            cost = work(case)["bytes"]
            size = case["buffers"] * case["groups"] * beams * case["outer"] * length * case["row"] * 4
            if size > 2 << 30:
                continue
        if cost <= most[op]:
            del case["name"]
            return case


# ------------------------------------------------------------------------------------------------------ the cases' lengths --
def _groups(case):
    """[(first row, rows, prefix length)]: rows as even as they go; ragged: lengths from the longest down to nothing."""
    rows, n, out, row = case["rows"], case["groups"], [], 0
    for g in range(n):
        take = rows // n + (g < rows % n)
        length = case["prefix"] if not case["ragged"] or n == 1 else case["prefix"] * (n - 1 - g) // (n - 1)
        out.append((row, take, length))
        row += take
    return out


def _tails(case):
    """Positions of every row's own, the new token's among them; 0: an idle row."""
    rows, tail = case["rows"], case["tail"]
    t = [tail if not case["ragged"] else 1 + (tail - 1) * ((37 * r + 11) % 64) // 63 for r in range(rows)]
    for r in range(case["idle"]):
        t[(5 * r + 1) % rows] = 0
    return t


def _vector(case):
    return case["count"] * case["row"] * torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()


def work(case):
    if case["op"] == "attention":
        h, hkv, d, tails = case["heads"], case["kv_heads"], case["dim"], _tails(case)
        live = sum(t > 0 for t in tails)
        keys = sum(n for n in tails) + sum(length for _, _, length in _groups(case))
        pairs = sum(tails) + sum(length * sum(tails[r] > 0 for r in range(r0, r0 + n)) for r0, n, length in _groups(case))
        return {"bytes": keys * hkv * d * 4 + live * h * d * 4, "flops": 4 * pairs * h * d}
    if case["op"] == "select":
        rows, size = case["groups"] * case["beams"], torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
        return {"bytes": rows * case["vocab"] * size + rows * 4 + case["groups"] * case["keep"] * 12, "flops": 3 * rows * case["vocab"]}
    sources = max(1, min(case["forks"] // 2, case["beams"] - case["forks"]))
    moved = case["buffers"] * case["groups"] * case["outer"] * _vector(case)
    return {"bytes": moved * (sources + case["forks"]), "flops": 0}


# ------------------------------------------------------------------------------------------------------------------ inputs --
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * int(seed) + 17)
    return g


def _attention_inputs(case, seed):
    g = _generator(seed)
    h, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    groups, tails = _groups(case), _tails(case)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=torch.float32).half()
    slots = torch.randperm(case["rows"], generator=g, device=DEV).tolist()
    kshape = (len(groups), hkv, max(case["prefix"], 1), d)
    oshape = (case["rows"], hkv, case["tail"] + 3, d)
    inp = {"q": rand(case["rows"], h, d) * 1.5, "pk": rand(*kshape), "pv": rand(*kshape), "k": rand(*oshape), "v": rand(*oshape)}
    inp["groups"] = [(r0, n, i, length, 0) for i, (r0, n, length) in enumerate(groups)]
    inp["slots"], inp["tails"] = slots, tails
    inp["row_slot"] = torch.tensor(slots, dtype=torch.int32, device=DEV)
    inp["row_pos"] = torch.tensor([t - 1 for t in tails], dtype=torch.int32, device=DEV)
    return inp


def _select_inputs(case, seed):
    g = _generator(seed)
    rows = case["groups"] * case["beams"]
    logits = (2.0 * torch.randn(rows, case["pitch"], generator=g, device=DEV)).to(DTYPES[case["dtype"]])
    if case["banned"]:
        out = torch.randperm(case["vocab"], generator=g, device=DEV)[:case["banned"]]
        logits[:, out] = -math.inf
    scores = torch.zeros(rows, device=DEV) if case["first"] else -20.0 - 4.0 * torch.rand(rows, generator=g, device=DEV)
    return logits[:, :case["vocab"]], scores


def _parents(case, seed):
    """[groups, beams]: the slot that each slot's next hypothesis comes from; one that survives keeps its slot."""
    rng = random.Random(31 * int(seed) + 7)
    sources = max(1, min(case["forks"] // 2, case["beams"] - case["forks"]))
    out = []
    for _ in range(case["groups"]):
        order = list(range(case["beams"]))
        rng.shuffle(order)
        ended, alive = order[:case["forks"]], order[case["forks"]:]
        row = list(range(case["beams"]))
        for i, b in enumerate(ended):
            row[b] = alive[i % sources]
        out.append(row)
    return out


def prepare(case, seed):
    if case["op"] == "attention":
        state = {"case": case, **_attention_inputs(case, seed)}
        state["out"] = torch.zeros_like(state["q"])
        # what the plain form reads from the host: the rows' lengths as index arrays
        state["own_len"] = torch.tensor(state["tails"], device=DEV)
        if own:
            from onebit_amd.beam import shared_prefix_workspace
            state["workspace"] = shared_prefix_workspace(state["groups"], case["rows"], case["heads"], case["kv_heads"], case["dim"],
                                                         case["tail"], device=DEV)
    elif case["op"] == "select":
        logits, scores = _select_inputs(case, seed)
        state = {"case": case, "logits": logits, "scores": scores}
        if own:
            from onebit_amd.beam import beam_select_workspace
            state["workspace"] = beam_select_workspace(logits.shape[0], case["vocab"], case["keep"], device=DEV)
    else:
        g = _generator(seed)
        shape = (case["groups"] * case["beams"], case["outer"], case["length"], case["row"])
        dt = DTYPES[case["dtype"]]
        state = {"case": case, "buffers": [torch.randn(shape, generator=g, device=DEV, dtype=dt) for _ in range(case["buffers"])],
                 "parents": torch.tensor(_parents(case, seed), dtype=torch.int32, device=DEV)}
    return state


# ------------------------------------------------------------------------------------------------------------------- a pass --
def _attention_plain(s):
    case, q = s["case"], s["q"]
    h, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    rep, scale = h // hkv, 1.0 / math.sqrt(d)
    out, tail = s["out"], case["tail"]
    for r0, n, slot, length, _ in s["groups"]:
        qg = q[r0:r0 + n].float().view(n, hkv, rep, d)
        idx = s["row_slot"][r0:r0 + n].long()
        lens = s["own_len"][r0:r0 + n]
        k, v = s["k"][idx, :, :tail].float(), s["v"][idx, :, :tail].float()                               # [n, hkv, tail, d]
        sc = (qg @ k.transpose(2, 3)) * scale                                                             # [n, hkv, rep, tail]
        sc = sc.masked_fill(torch.arange(tail, device=DEV) >= lens[:, None, None, None], -math.inf)
        m = sc.amax(-1)
        if length:
            pk, pv = s["pk"][slot, :, :length].float(), s["pv"][slot, :, :length].float()                 # [hkv, length, d]
            qp = qg.transpose(0, 1).reshape(hkv, n * rep, d)
            sp = ((qp @ pk.transpose(1, 2)) * scale).view(hkv, n, rep, length).transpose(0, 1)            # [n, hkv, rep, length]
            m = torch.maximum(m, sp.amax(-1))
        p = torch.exp(sc - m[..., None])
        total, o = p.sum(-1), p @ v
        if length:
            p = torch.exp(sp - m[..., None])
            total = total + p.sum(-1)
            o = o + (p.transpose(0, 1).reshape(hkv, n * rep, length) @ pv).view(hkv, n, rep, d).transpose(0, 1)
        o = (o / total[..., None]).reshape(n, h, d).to(q.dtype)
        out[r0:r0 + n] = torch.where((lens > 0)[:, None, None], o, out[r0:r0 + n])
    return out


def _descending_keys(x):
    """Whole numbers that order like ``x`` and, among equal values, put the lower index first."""
    bits = (x.float() + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
    return (order << 32) - torch.arange(x.shape[-1], device=x.device)


def _select_plain(s):
    case, logits, scores = s["case"], s["logits"], s["scores"]
    beams, keep, v = case["beams"], case["keep"], case["vocab"]
    x = logits.double()
    m = x.amax(-1, keepdim=True)
    lse = m + torch.log(torch.exp(x - m).sum(-1, keepdim=True))
    near = min(keep, v)
    tokens = torch.topk(_descending_keys(logits), near, dim=-1).indices                                   # a row's best, in order
    val = scores.double()[:, None] + (torch.gather(x, 1, tokens) - lse)
    val = torch.where(torch.isnan(val), -math.inf, val).view(-1, beams * near)
    val, at = torch.sort(val, dim=-1, descending=True, stable=True)
    val, at = val[:, :keep], at[:, :keep]
    tok = torch.gather(tokens.view(-1, beams * near), 1, at)
    none = val == -math.inf
    return [val.float(), torch.where(none, -1, at // near).int(), torch.where(none, -1, tok).int()]


def _reorder_plain(s):
    case = s["case"]
    first, end, n = case["first"], case["first"] + case["count"], case["groups"] * case["beams"]
    base = torch.arange(0, n, case["beams"], device=DEV)[:, None]
    src = (s["parents"].long() + base).view(-1)
    for b in s["buffers"]:
        b[:, :, first:end] = b[src, :, first:end]
    return s["buffers"]


def run(state):
    case = state["case"]
    if not own:
        return {"attention": _attention_plain, "select": _select_plain, "reorder": _reorder_plain}[case["op"]](state)
    from onebit_amd.beam import beam_select, reorder_slots, shared_prefix_attention
    if case["op"] == "attention":
        return shared_prefix_attention(state["q"], state["pk"], state["pv"], state["k"], state["v"], state["groups"], state["row_slot"],
                                       state["row_pos"], max_own=case["tail"], out=state["out"], workspace=state["workspace"])
    if case["op"] == "select":
        return list(beam_select(state["logits"], state["scores"], case["beams"], case["keep"], workspace=state["workspace"]))
    reorder_slots(state["buffers"], state["parents"], first=case["first"], count=case["count"])
    return state["buffers"]


# -------------------------------------------------------------------------------------------------------- 64-bit definitions --
def _attention_exact(case, seed):
    s = _attention_inputs(case, seed)
    h, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(case["rows"], h, d, dtype=torch.float64, device=DEV)
    for r0, n, slot, length, _ in s["groups"]:
        for kv in range(hkv):
            heads = slice(kv * (h // hkv), (kv + 1) * (h // hkv))
            pk, pv = s["pk"][slot, kv, :length].double(), s["pv"][slot, kv, :length].double()
            for r in range(r0, r0 + n):
                t = s["tails"][r]
                if not t:
                    continue
                k = torch.cat([pk, s["k"][s["slots"][r], kv, :t].double()])
                v = torch.cat([pv, s["v"][s["slots"][r], kv, :t].double()])
                w = torch.softmax(torch.mm(s["q"][r, heads].double(), k.t()) / math.sqrt(d), dim=-1)
                out[r, heads] = torch.mm(w, v)
    return out


def _select_exact(case, seed):
    logits, scores = _select_inputs(case, seed)
    beams, keep = case["beams"], case["keep"]
    val, beam, tok = [], [], []
    for g in range(case["groups"]):
        x = logits[g * beams:(g + 1) * beams].double()
        flat = (scores[g * beams:(g + 1) * beams].double()[:, None] + torch.log_softmax(x, dim=-1)).reshape(-1)
        flat = torch.nan_to_num(flat, nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        best, at = torch.sort(flat, descending=True, stable=True)
        best, at = best[:keep], at[:keep]
        none = best == -math.inf
        val.append(best)
        beam.append(torch.where(none, -1, at // case["vocab"]))
        tok.append(torch.where(none, -1, at % case["vocab"]))
    pad = lambda rows, value: torch.stack([torch.nn.functional.pad(r, (0, keep - r.numel()), value=value) for r in rows])
    return [pad(val, -math.inf), pad(beam, -1).int(), pad(tok, -1).int()]


def _reorder_exact(case, seed):
    s = prepare(case, seed)
    first, end, beams = case["first"], case["first"] + case["count"], case["beams"]
    out = []
    for b in s["buffers"]:
        moved = b.clone()
        for g, row in enumerate(_parents(case, seed)):
            for i, p in enumerate(row):
                moved[g * beams + i, :, first:end] = b[g * beams + p, :, first:end]
        out.append(moved)
    return out


def exact(case, seed):
    if case["op"] == "attention":
        # (a product for every row and key head: two microseconds' worth of arithmetic each, some tens of launch overhead)
        return _attention_exact(case, seed)
    return _select_exact(case, seed) if case["op"] == "select" else _reorder_exact(case, seed)
