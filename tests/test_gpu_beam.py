"""Beam search's operators against their definitions in 64 bits."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from onebit_amd.beam import beam_select, beam_select_workspace, reorder_slots, shared_prefix_attention, shared_prefix_workspace

F16, F64 = torch.float16, torch.float64


# ------------------------------------------------------------------------------------------------ attention over a shared prefix --
def _case(lens, rows, own, H, hkv, D, seed=0, one_cache=False, idle=(), scale=1.0):
    """Groups of ``rows[g]`` rows with prefixes of ``lens[g]``, row r with own[r] positions of its own.  Everything that no row may read is NaN."""
    g = torch.Generator().manual_seed(seed)
    n, G = sum(rows), len(lens)
    rand = lambda *s: (scale * torch.randn(*s, generator=g)).to(F16)
    nan = lambda *s: torch.full(s, math.nan, dtype=F16)
    first = [l if one_cache else 0 for l in lens]
    longest = max(max(lens), 1)
    own_len = max([longest + max(own) if one_cache else max(own)]) + 2
    slots = n + (G if one_cache else 0)
    order = torch.randperm(slots, generator=g).tolist()
    k, v = nan(slots, hkv, own_len, D), nan(slots, hkv, own_len, D)
    pk, pv = (k, v) if one_cache else (nan(G, hkv, longest, D), nan(G, hkv, longest, D))
    groups, row_slot, row_pos, r = [], [], [], 0
    for gi, (l, m) in enumerate(zip(lens, rows)):
        ps = order[n + gi] if one_cache else gi
        pk[ps, :, :l], pv[ps, :, :l] = rand(hkv, l, D), rand(hkv, l, D)
        groups.append((r, m, ps, l, first[gi]))
        for i in range(r, r + m):
            k[order[i], :, first[gi]:first[gi] + own[i]], v[order[i], :, first[gi]:first[gi] + own[i]] = rand(hkv, own[i], D), rand(hkv, own[i], D)
            row_slot.append(order[i])
            row_pos.append(first[gi] + own[i] - 1)
        r += m
    for j, i in enumerate(idle):
        if j % 2:
            row_slot[i] = -1 if j % 4 == 1 else slots
        else:
            row_pos[i] = -1 if j % 4 == 0 else own_len
    idle = set(idle) | {i for i, p in enumerate(row_pos) if p < 0}                  # (no position at all is an idle row, by definition)
    dev = lambda t: t.cuda()
    out = dict(q=dev(rand(n, H, D)), pk=dev(pk), pv=dev(pv), k=dev(k), v=dev(v), groups=groups, own=own, idle=idle,
               row_slot=torch.tensor(row_slot, dtype=torch.int32).cuda(), row_pos=torch.tensor(row_pos, dtype=torch.int32).cuda(), slots=row_slot)
    if one_cache:
        out["pk"], out["pv"] = out["k"], out["v"]
    return out


def _call(c, **kw):
    return shared_prefix_attention(c["q"], c["pk"], c["pv"], c["k"], c["v"], c["groups"], c["row_slot"], c["row_pos"], max_own=kw.pop("max_own", max(c["own"])), **kw)


def _reference(c):
    """Outputs in 64 bits and how far the kernel's may be.  Weights are rounded to fp16 (2^-11 each, on numerator and denominator alike: 2^-11 (A + |o|) with
    A the weighted mean of |v|; below 2^-14 of the largest by 2^-25 of it), the output is (2^-11 |o|, 2^-25).  fp32: a score is off by (D + 4) 2^-24 times the
    sum of its terms' sizes, its weight by as much; sums of n weights and values by n 2^-24."""
    n, H, D = c["q"].shape
    hkv = c["k"].shape[1]
    out, tol = torch.zeros(n, H, D, dtype=F64, device="cuda"), torch.zeros(n, H, D, dtype=F64, device="cuda")
    for r0, m, slot, l, first in c["groups"]:
        for r in range(r0, r0 + m):
            if r in c["idle"]:
                continue
            e = first + c["own"][r]
            k = torch.cat([c["pk"][slot, :, :l], c["k"][c["slots"][r], :, first:e]], dim=1).double().repeat_interleave(H // hkv, 0)
            v = torch.cat([c["pv"][slot, :, :l], c["v"][c["slots"][r], :, first:e]], dim=1).double().repeat_interleave(H // hkv, 0)
            if k.shape[1] == 0:
                continue
            q = c["q"][r].double()[:, None]
            w = torch.softmax((q * k).sum(-1) / math.sqrt(D), -1)[..., None]
            o, a = (w * v).sum(1), (w * v.abs()).sum(1)
            size = ((q.abs() * k.abs()).sum(-1) / math.sqrt(D)).amax(-1)[:, None]
            keys = k.shape[1]
            eps = 2 * ((D + 8) * 2.0 ** -24 * size + (keys + 64) * 2.0 ** -24)
            out[r] = o
            tol[r] = (2.0 ** -11 * (a + o.abs()) + 2.0 ** -11 * o.abs() + keys * 2.0 ** -25 * v.abs().amax(1)) * 1.002 + eps * a + 2.0 ** -25
    return out, tol


def _check(c, y):
    ref, tol = _reference(c)
    live = [r for r in range(y.shape[0]) if r not in c["idle"]]
    assert torch.isfinite(y[live].float()).all()
    err = ((y.double() - ref).abs() - tol)[live]
    assert err.max() <= 0, f"{err.max().item()} beyond the bound"


LENS = [0, 1, 5, 31, 32, 33, 127, 128, 129, 300, 1000]


@pytest.mark.parametrize("D", [128, 64, 96, 40, 8])
@pytest.mark.parametrize("length", LENS)
def test_lengths(D, length):
    _check(c := _case([length], [3], [1, 40, 7], 4, 2, D, seed=length + D), _call(c))


@pytest.mark.parametrize("H, hkv", [(1, 1), (8, 8), (8, 1), (12, 4), (40, 2), (33, 1)])
@pytest.mark.parametrize("rows", [1, 2, 9, 17, 33, 70])
def test_heads_and_rows(H, hkv, rows):
    own = [1 + (11 * r) % 37 for r in range(rows)]
    _check(c := _case([260], [rows], own, H, hkv, 64, seed=rows), _call(c))


@pytest.mark.parametrize("own", [0, 1, 32, 33, 127, 128, 129, 700])
def test_own_positions(own):
    _check(c := _case([50, 0], [2, 2], [own, max(own - 1, 0), own, 3], 4, 4, 128, seed=own), _call(c, max_own=max(own, 3)))


@pytest.mark.parametrize("H, hkv, rows, length, own", [(8, 8, 40, 100, 300), (16, 2, 20, 200, 300), (16, 2, 5, 300, 900), (16, 2, 5, 5000, 900), (64, 2, 9, 700, 1),
                                                       (4, 4, 64, 3000, 20), (24, 1, 7, 2100, 130), (2, 2, 64, 0, 200), (8, 1, 3, 4000, 600)])
def test_many_queries_and_long_own_positions(H, hkv, rows, length, own):
    """16, 64 and 128 queries a workgroup; own positions that outweigh the prefix, that are split, that are few."""
    lens, n = [length, length // 3], [rows - 1, 1]
    own = [1 + (own * ((7 * r) % rows)) // rows for r in range(rows - 1)] + [own]
    _check(c := _case(lens, n, own, H, hkv, 128 if H != 24 else 72, seed=rows, idle=(1,)), _call(c))


@pytest.mark.parametrize("one_cache", [False, True])
def test_ragged_groups_and_idle_rows(one_cache):
    lens, rows = [515, 64, 0, 1, 130], [5, 1, 3, 2, 4]
    own = [3, 90, 1, 17, 33, 260, 5, 4, 64, 65, 2, 9, 128, 129, 31]
    c = _case(lens, rows, own, 8, 2, 128, seed=3, one_cache=one_cache, idle=(1, 6, 7, 14))
    out = torch.full_like(c["q"], 7.0)
    y = _call(c, out=out)
    assert y is out
    _check(c, y)
    assert all((y[r] == 7.0).all() for r in c["idle"])
    again = _call(c)
    assert all((again[r] == 0).all() for r in c["idle"])
    live = [r for r in range(15) if r not in c["idle"]]
    assert torch.equal(again[live], y[live])


def test_more_groups_than_one_launch_takes():
    lens, rows = [(37 * i) % 200 for i in range(150)], [1 + i % 2 for i in range(150)]
    own = [1 + (13 * r) % 50 for r in range(sum(rows))]
    _check(c := _case(lens, rows, own, 2, 1, 64, seed=8), _call(c))


def test_row_without_any_key_gets_zeros():
    c = _case([0, 4], [1, 1], [0, 1], 2, 2, 64, one_cache=False)
    c["groups"] = [(0, 1, 0, 0, 2), (1, 1, 1, 4, 0)]                 # row 0 sits at position 0, its own positions begin at 2
    c["row_pos"] = torch.tensor([0, 0], dtype=torch.int32, device="cuda")
    y = _call(c, out=torch.full_like(c["q"], 7.0))
    assert (y[0] == 0).all() and torch.isfinite(y[1].float()).all() and (y[1] != 0).any()


def test_positions_beyond_the_bound_are_left_out():
    c = _case([20], [2], [40, 300], 2, 2, 64, seed=5)
    y = _call(c, max_own=200)
    c["own"] = [40, 200]
    _check(c, y)


def test_no_prefix_cache_and_default_arguments():
    c = _case([0], [4], [5, 1, 200, 64], 4, 4, 64)
    c["slots"] = list(range(4))
    k = torch.randn(4, 4, 210, 64, device="cuda").to(F16)
    c["k"], c["v"] = k, torch.randn_like(k)
    y = shared_prefix_attention(c["q"], None, None, c["k"], c["v"], [(0, 4, 0, 0, 0)], None, c["row_pos"])
    _check(c, y)


def test_output_scaling():
    c = _case([70], [3], [5, 1, 20], 4, 4, 64, seed=9)
    h = torch.rand(4 * 64, device="cuda").to(F16) + 0.5
    assert torch.equal(_call(c, h_next=h), _call(c) * h.view(4, 64))
    for rows, length, own in ((3, 500, 20), (40, 500, 20), (40, 50, 200), (40, 5000, 600)):          # every form writes its outputs itself
        c = _case([length], [rows], [own] * rows, 4, 4, 64, seed=rows)
        assert torch.equal(_call(c, h_next=h), _call(c) * h.view(4, 64))


def test_large_scores_and_one_far_maximum():
    """Scores of hundreds: the maximum lies far behind the first keys, and all other weights underflow."""
    c = _case([600], [3], [40, 1, 9], 2, 2, 64, seed=2, scale=6.0)
    _check(c, _call(c))


@pytest.mark.parametrize("H, hkv, rows, length, own", [(4, 4, 8, 1500, 70), (2, 2, 33, 1500, 70), (16, 2, 20, 9000, 70), (4, 4, 8, 200, 70), (2, 2, 33, 0, 700), (16, 2, 40, 0, 1300),
                                                       (2, 2, 64, 600, 1500), (64, 2, 9, 40000, 40)])
@pytest.mark.parametrize("high", [11, 17, 40])
def test_a_maximum_that_moves_late(H, hkv, rows, length, own, high):
    """Every query's largest score stands at a place of its own behind many small ones, so far above them that the running maximum has to move there: all 32 places of a step
    of keys, in prefix and own keys, in all forms."""
    c = _case([length], [rows], [own - (r % 3) for r in range(rows)], H, hkv, 64, seed=high, scale=0.05)
    n = H // hkv
    scores = high * math.log(2.0) * 8.0                                 # (times 1 / sqrt(64), log2 e: `high` in powers of two)
    q = c["q"]
    for r in range(rows):
        for h in range(H):
            q[r, h, (5 * r + h) % 32] = math.sqrt(scores)
    for i in range(32):
        if length:
            c["pk"][0, :, length - 33 * i - 5 if length > 1100 else length - 5 * i - 3, i] = math.sqrt(scores)
        else:
            for s in c["slots"]:
                c["k"][s, :, own - 19 * i - 4, i] = math.sqrt(scores)
    assert n * hkv == H
    _check(c, _call(c))


@pytest.mark.parametrize("H, hkv, rows, length, own, D", [(4, 4, 8, 200, 70, 64), (4, 4, 8, 1501, 70, 128), (2, 2, 33, 1509, 70, 64), (2, 2, 33, 1571, 70, 40), (16, 2, 20, 4001, 70, 128),
                                                          (2, 2, 64, 1541, 1500, 64), (64, 1, 64, 8301, 37, 128), (64, 1, 64, 8193, 37, 80), (16, 2, 40, 0, 1299, 64), (40, 40, 64, 999, 9, 64)])
def test_infinities_and_nan_in_values(H, hkv, rows, length, own, D):
    """A value that is infinite or NaN makes that column of its rows infinite or NaN and no other, also in the last row of a prefix or of a row's own positions, in all
    forms: no place behind a range takes part in the products."""
    c = _case([length], [rows], [own] * rows, H, hkv, D, seed=length + D, scale=0.5)
    col = dict(zip((3, 7, 11), (math.inf, -math.inf, math.nan)))
    for d, bad in col.items():
        if length:
            c["pv"][0, :, length - 1, d] = bad
        c["v"][c["slots"][0], :, own - 1, d + 1] = bad
    y = _call(c)
    for d, bad in col.items():
        same = torch.isnan if math.isnan(bad) else lambda t, bad=bad: t == bad
        if length:
            assert same(y[:, :, d]).all(), (d, bad)
            c["pv"][0, :, length - 1, d] = 0
        assert same(y[0, :, d + 1]).all(), (d, bad)
        c["v"][c["slots"][0], :, own - 1, d + 1] = 0
    clean = _call(c)
    ref, tol = _reference(c)
    for d in col:
        if length:
            y[:, :, d] = clean[:, :, d]
        y[0, :, d + 1] = clean[0, :, d + 1]
    assert torch.isfinite(y).all() and ((y.double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("D", [128, 64, 80, 40])
@pytest.mark.parametrize("length", [8192, 8301])
def test_blocks_of_128_queries(D, length):
    """Tiles brought by DMA, whole and padded heads, a last tile that is not full, a second group without a prefix."""
    _check(c := _case([length, 0], [63, 1], [1 + (7 * r) % 40 for r in range(64)], 64, 1, D, seed=D, idle=(5,)), _call(c))


@pytest.mark.parametrize("H, hkv, rows, length, own", [(4, 4, 40, 2000, 50), (64, 1, 64, 8200, 20), (4, 4, 40, 2000, 500), (2, 1, 6, 20000, 30)])
def test_every_replay_of_a_graph_is_the_eager_call(H, hkv, rows, length, own):
    c = _case([length], [rows], [1 + (own * ((5 * r) % rows)) // rows for r in range(rows)], H, hkv, 128, seed=rows)
    ws = shared_prefix_workspace(c["groups"], rows, H, hkv, 128, own)
    out = torch.zeros_like(c["q"])
    _call(c, out=out, workspace=ws, max_own=own)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _call(c, out=out, workspace=ws, max_own=own)
    for i in range(3):
        c["q"].copy_(torch.randn_like(c["q"]))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        y = out.clone()
        assert torch.equal(_call(c, max_own=own), y)
    _check(c, y)


def test_offsets_beyond_32_bits():
    """A prefix in the last slot of a cache whose slots hold 2 GiB each, and own positions far inside a slot."""
    long = (1 << 23) + 40
    cache = torch.empty(3, 1, long, 128, dtype=F16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    far = torch.randn(300, 128, generator=g, device="cuda").to(F16)
    cache[2, 0, :300] = far
    cache[1, 0, long - 40:] = far[:40]
    q = torch.randn(1, 2, 128, generator=g, device="cuda").to(F16)
    pos = torch.tensor([long - 1], dtype=torch.int32, device="cuda")
    y = shared_prefix_attention(q, cache, cache, cache, cache, [(0, 1, 2, 300, long - 40)], torch.tensor([1], dtype=torch.int32, device="cuda"), pos, max_own=40)
    keys = torch.cat([far, far[:40]]).double()
    w = torch.softmax(q[0].double() @ keys.t() / math.sqrt(128), -1)
    ref, a = w @ keys, w @ keys.abs()
    assert ((y[0].double() - ref).abs() <= 2.0 ** -11 * (a + 2 * ref.abs()) * 1.01 + 1e-5 * a).all()


def test_replayed_in_a_graph_with_new_positions():
    c = _case([150], [4], [60, 60, 60, 60], 4, 2, 128, seed=6)
    ws = shared_prefix_workspace(c["groups"], 4, 4, 2, 128, 60)
    out = torch.zeros_like(c["q"])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _call(c, out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _call(c, out=out, workspace=ws)
    for own in ([1, 2, 3, 4], [60, 60, 60, 60], [33, 1, 59, 32]):
        c["own"] = own
        c["row_pos"].copy_(torch.tensor([n - 1 for n in own], dtype=torch.int32))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        y = out.clone()
        _check(c, y)
        assert torch.equal(_call(c, max_own=60), y)


def test_one_workspace_for_calls_of_many_sizes_in_turn():
    big = shared_prefix_workspace([(0, 70, 0, 4000, 0)], 70, 40, 40, 128, 900)
    for seed, (l, n, H, hkv, D) in enumerate([(300, 3, 4, 4, 64), (20, 9, 8, 2, 128), (1000, 2, 2, 1, 40), (300, 3, 4, 4, 64)]):
        c = _case([l], [n], [1 + 5 * i for i in range(n)], H, hkv, D, seed=seed)
        y = _call(c, workspace=big)
        _check(c, y)
        assert torch.equal(y, _call(c))


def test_scratch_contents_are_of_no_account_but_for_the_counters():
    for rows, length, own in ((4, 900, 20), (40, 900, 300), (6, 5000, 900)):
        c = _case([length], [rows], [own] * rows, 4, 4, 128, seed=rows)
        ws = shared_prefix_workspace(c["groups"], rows, 4, 4, 128, own)
        y = _call(c, workspace=ws)
        ws[4 * 16384:] = 255                                        # NaN, as floats
        z = _call(c, workspace=ws)
        assert torch.equal(y, z) and not ws[:4 * 16384].any()
        _check(c, z)


def test_the_same_bits_every_time():
    for rows, H, hkv, length, own in ((5, 8, 8, 3000, 100), (24, 8, 2, 2000, 700), (64, 8, 8, 900, 60)):
        c = _case([length, length // 2], [rows - 2, 2], [1 + (own * ((7 * r) % rows)) // rows for r in range(rows)], H, hkv, 64, seed=rows)
        ws = shared_prefix_workspace(c["groups"], rows, H, hkv, 64, own)
        y = _call(c, workspace=ws)
        _check(c, y)
        assert all(torch.equal(_call(c, workspace=ws), y) for _ in range(50))


def test_streams_at_the_same_time():
    """Calls on two streams, each with a workspace of its own."""
    cases = [_case([1500], [6], [40 + i] * 6, 8, 8, 128, seed=i) for i in range(2)]
    want = [_call(c) for c in cases]
    ws = [shared_prefix_workspace(c["groups"], 6, 8, 8, 128, max(c["own"])) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(_call(cases[i], workspace=ws[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for ys, w in zip(got, want) for y in ys)


def test_two_graphs_with_one_workspace_replayed_in_turn():
    cases = [_case([700 + 900 * i], [3 + 4 * i], [50] * (3 + 4 * i), 4, 4, 64, seed=i) for i in range(2)]
    ws = shared_prefix_workspace(cases[1]["groups"], 7, 4, 4, 64, 50)
    outs, graphs = [torch.zeros_like(c["q"]) for c in cases], []
    for c, o in zip(cases, outs):
        _call(c, out=o, workspace=ws)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            _call(c, out=o, workspace=ws)
    for _ in range(3):
        for c, o, g in zip(cases, outs, graphs):
            o.zero_()
            g.replay()
        torch.cuda.synchronize()
        for c, o in zip(cases, outs):
            _check(c, o)


def test_thousands_of_rows():
    """More rows than the counters count: the launches for many."""
    lens, rows = [(53 * i) % 400 for i in range(600)], [1 + i % 9 for i in range(600)]
    own = [1 + (13 * r) % 40 for r in range(sum(rows))]
    assert sum(rows) * 8 > 16384
    _check(c := _case(lens, rows, own, 8, 8, 40, seed=8), _call(c))


def test_attention_python_refusals():
    c = _case([700], [3], [5, 1, 20], 4, 4, 64)
    bad = [dict(q=c["q"].float()), dict(q=c["q"][:, :, :32]), dict(k=c["k"].float()), dict(pk=None), dict(row_pos=c["row_pos"].long()), dict(row_pos=c["row_pos"][:2]),
           dict(groups=[(0, 3, 5, 700, 0)]), dict(groups=[(0, 2, 0, 700, 0)]), dict(row_slot=c["row_slot"].cpu()), dict(v=c["v"][:, :2])]
    for b in bad:
        with pytest.raises(ValueError):
            _call({**c, **b})
    for b in (dict(out=c["q"]), dict(out=c["q"].float()), dict(h_next=c["q"][0, 0]), dict(workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(ValueError):
            _call(c, **b)


def test_an_output_beside_its_inputs_but_not_over_them():
    c = _case([700], [3], [5, 1, 20], 4, 4, 64)
    want = _call(c)
    both = torch.zeros(6, 4, 64, dtype=F16, device="cuda")
    both[:3] = c["q"]
    c["q"] = both[:3]
    assert torch.equal(_call(c, out=both[3:]), want) and torch.equal(both[3:], want)
    for out in (both[1:4], both[2:5], c["k"].view(-1)[40:40 + 768].view(3, 4, 64), c["pv"].view(-1)[-768:].view(3, 4, 64)):
        with pytest.raises(ValueError, match="overlap"):
            _call(c, out=out)
    assert torch.equal(_call(c), want)


# ------------------------------------------------------------------------------------------------------- the choice of hypotheses --
def _best(logits, scores, beams, keep):
    """The definition on the CPU: every continuation of every hypothesis, in the documented order."""
    x = logits.double().cpu()
    s = scores.double().cpu()
    rows, V = x.shape
    val, beam, tok = [], [], []
    for g in range(rows // beams):
        lse = torch.logsumexp(x[g * beams:(g + 1) * beams], -1)
        v = s[g * beams:(g + 1) * beams, None] + (x[g * beams:(g + 1) * beams] - lse[:, None])
        v = torch.where(torch.isnan(v), -math.inf, v)
        cand = []
        for b in range(beams):
            order = torch.sort(x[g * beams + b].nan_to_num(nan=-math.inf) + 0.0, descending=True, stable=True).indices[:keep + 1].tolist()
            cand += [(-v[b, t].item(), b, i, t) for i, t in enumerate(order) if v[b, t] > -math.inf]
        cand = sorted(cand)[:keep]
        cand += [(math.inf, -1, 0, -1)] * (keep - len(cand))
        val.append([-c[0] for c in cand])
        beam.append([c[1] for c in cand])
        tok.append([c[3] for c in cand])
    return torch.tensor(val, dtype=F64), torch.tensor(beam, dtype=torch.int32), torch.tensor(tok, dtype=torch.int32)


def _check_select(logits, scores, beams, keep, **kw):
    v, b, t = beam_select(logits, scores, beams, keep, **kw)
    rv, rb, rt = _best(logits, scores, beams, keep)
    assert torch.equal(b.cpu(), rb) and torch.equal(t.cpu(), rt)
    fin = torch.isfinite(rv)
    assert torch.equal(torch.isfinite(v.cpu()), fin)
    # the value: half a step of fp32, and the logarithm of a sum whose terms are off by 2^-23
    assert ((v.cpu().double() - rv)[fin].abs() <= 2.0 ** -24 * rv[fin].abs() + 2.0 ** -22).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("groups, beams, vocab, keep", [(1, 1, 1, 1), (1, 1, 1, 4), (2, 3, 5, 8), (1, 4, 512, 8), (3, 2, 2047, 4), (2, 8, 2048, 16), (1, 5, 2049, 10),
                                                        (4, 4, 32000, 8), (1, 32, 4099, 64), (65, 1, 300, 2), (1, 2, 128256, 4), (2, 16, 50257, 32)])
def test_choice(dtype, groups, beams, vocab, keep):
    g = torch.Generator(device="cuda").manual_seed(vocab + beams)
    logits = (2 * torch.randn(groups * beams, vocab, generator=g, device="cuda")).to(dtype)
    scores = -20 - 3 * torch.rand(groups * beams, generator=g, device="cuda")
    _check_select(logits, scores, beams, keep)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("keep", [1, 7, 64])
def test_ties_go_to_the_lowest_beam_and_token(dtype, keep):
    g = torch.Generator(device="cuda").manual_seed(keep)
    row = torch.randint(-1, 3, (1, 5001), generator=g, device="cuda").to(dtype)
    logits = row.repeat(6, 1)                                       # equal hypotheses: every value occurs in each of them, many times
    _check_select(logits, torch.full((6,), -3.0, device="cuda"), 3, keep)
    _check_select(torch.zeros(4, 5001, dtype=dtype, device="cuda"), torch.zeros(4, device="cuda"), 4, keep)


@pytest.mark.parametrize("vocab, beams, keep, banned", [(512, 32, 64, 0), (512, 32, 64, 300), (32000, 32, 64, 10666), (9001, 2, 64, 0), (50257, 32, 64, 0), (520, 3, 64, 500)])
@pytest.mark.parametrize("values", ["many", "few"])
def test_more_candidates_than_a_list_holds(vocab, beams, keep, banned, values):
    """Many kept next to a chunk's lanes, few distinct values, banned tokens in runs: the search for a threshold, lists that the pick chooses from first."""
    g = torch.Generator(device="cuda").manual_seed(vocab + keep)
    x = 2 * torch.randn(2 * beams, vocab, generator=g, device="cuda")
    if values == "few":
        x = (x * 2).round() / 2
        x[:, ::7] *= -0.0                                            # zeros of both signs are equal logits
    x[:, vocab // 3:vocab // 3 + banned] = -math.inf
    scores = -10 - 2 * torch.rand(2 * beams, generator=g, device="cuda")
    _check_select(x.half(), scores, beams, keep)
    _check_select(x, scores, beams, keep)


@pytest.mark.parametrize("vocab", [600000, (1 << 20) - 3])
@pytest.mark.parametrize("values", ["many", "few"])
def test_more_lists_than_the_pick_chooses_from_first(vocab, values):
    """32 hypotheses of 74 and of 128 chunks each: every place of every list is looked at."""
    g = torch.Generator(device="cuda").manual_seed(vocab % 97)
    x = 2 * torch.randn(32, vocab, generator=g, device="cuda")
    if values == "few":
        x = x.round()
    x[:, :vocab // 3] = -math.inf
    _check_select(x.half(), -10 - 2 * torch.rand(32, generator=g, device="cuda"), 32, 64)


def test_equal_rows_at_every_alignment_have_equal_values():
    """Rows of an odd pitch begin at all alignments; the sums must not depend on it, or ties between beams would break."""
    g = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.zeros(8, 4001, dtype=F16, device="cuda")
    wide[:, :3999] = (3 * torch.randn(1, 3999, generator=g, device="cuda")).to(F16)
    _check_select(wide[:, :3999], torch.zeros(8, device="cuda"), 8, 16)
    _check_select(wide[:, 1:4000], torch.zeros(8, device="cuda"), 8, 16)


def test_dead_hypotheses_banned_tokens_and_broken_rows():
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = torch.randn(24, 3000, generator=g, device="cuda")
    scores = -torch.rand(24, generator=g, device="cuda")
    scores[1] = -math.inf                                           # a dead hypothesis
    scores[4:8] = -math.inf                                         # a group of them
    logits[8, 5] = math.nan
    logits[9, 2999] = math.inf
    logits[10] = -math.inf
    logits[12:16, 7:] = -math.inf                                   # seven tokens allowed
    logits[16:20] = -math.inf
    logits[16, 2500] = 1.0                                          # a single continuation
    scores[20] = -1e9                                               # values that 64 bits no longer tell apart
    logits[20] = logits[20] * 1e-9
    scores[21:24] = -math.inf
    _check_select(logits, scores, 4, 40)


def test_far_below_the_maximum():
    """A peaked row: nearly all of its terms vanish next to the largest."""
    g = torch.Generator(device="cuda").manual_seed(3)
    logits = 30 * torch.randn(8, 10007, generator=g, device="cuda")
    logits[:, 77] = 300.0
    _check_select(logits, torch.zeros(8, device="cuda"), 4, 20)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("kind", ["normal", "narrow", "wide", "equal", "two"])
def test_the_logarithm_of_a_row_s_sum(kind, dtype):
    """How far values are from 64 bits.  A term e^d, d = x - max, is off by 2^-24 |d| twice (the difference and its product with log2 e, rounded), by 2^-26 |d| (the constant) and by 2^-23
    (the exponential), so the logarithm of the sum by 2^-23 (1 + 9/8 mean |d|), the mean over the row's probabilities."""
    g = torch.Generator(device="cuda").manual_seed(7)
    n, vocab = 40, 32003
    x = torch.randn(n, vocab, generator=g, device="cuda")
    if kind == "equal":
        x = torch.linspace(-9, 0, n, device="cuda")[:, None].repeat(1, vocab)
    elif kind == "two":                                              # half of the row at each of two places: every term of a half is off by the same
        x = torch.where(x < 0, torch.linspace(-20, 0, n, device="cuda")[:, None], torch.linspace(-5, -4, n, device="cuda")[:, None])
    else:
        x = x * {"normal": 2.0, "narrow": 0.1, "wide": 12.0}[kind]
    x[:, 0] = x.amax(1) + torch.linspace(0, 9, n, device="cuda")
    x = x.to(dtype)
    d = x.double()
    lse, top = torch.logsumexp(d, -1), d.amax(-1)
    scores = (lse - top).float()                                     # the best value is then nearly zero, where fp32 shows small errors
    v = beam_select(x, scores, 1, 1)[0][:, 0].double()
    ref = scores.double() + (top - lse)
    tol = 2.0 ** -23 * (1 + 9 / 8 * ((top[:, None] - d) * torch.softmax(d, -1)).sum(-1)) * 1.001
    err = (v - ref).abs()
    assert (err <= tol).all()


def test_select_in_a_graph_and_with_a_kept_workspace():
    ws = beam_select_workspace(16, 40000, 64)
    g = torch.Generator(device="cuda").manual_seed(4)
    logits, scores = torch.randn(8, 9001, generator=g, device="cuda"), torch.rand(8, generator=g, device="cuda")
    _check_select(logits, scores, 4, 8, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = beam_select(logits, scores, 4, 8, workspace=ws)
    for seed in range(3):
        logits.copy_(torch.randn(8, 9001, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        rv, rb, rt = _best(logits, scores, 4, 8)
        assert torch.equal(out[1].cpu(), rb) and torch.equal(out[2].cpu(), rt)
        _check_select(logits, scores, 2, 5, workspace=ws)           # the workspace serves another call in between


def test_select_gives_the_same_bits_every_time_on_any_stream():
    g = torch.Generator(device="cuda").manual_seed(5)
    inputs = [(torch.randn(b * n, v, generator=g, device="cuda"), -torch.rand(b * n, generator=g, device="cuda"), b) for n, b, v in ((1, 4, 32000), (2, 8, 9001), (64, 4, 3000))]
    ws = [beam_select_workspace(x.shape[0], x.shape[1], 2 * b) for x, _, b in inputs]
    want = [[t.clone() for t in beam_select(x, s, b, 2 * b)] for x, s, b in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for i, (x, s, b) in enumerate(inputs):
            with torch.cuda.stream(streams[i]):
                got.append((i, beam_select(x, s, b, 2 * b, workspace=ws[i])))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i, y in got for a, b in zip(y, want[i]))
    assert not any(w[:4 * 4096].any() for w in ws)


def test_select_many_groups():
    g = torch.Generator(device="cuda").manual_seed(6)
    _check_select(torch.randn(5000, 33, generator=g, device="cuda"), -torch.rand(5000, generator=g, device="cuda"), 1, 3)


def test_select_python_refusals():
    x, s = torch.zeros(8, 100, device="cuda"), torch.zeros(8, device="cuda")
    for args in ((x, s, 3, 4), (x, s, 4, 0), (x, s, 4, 65), (x, s.double(), 4, 8), (x.t(), s, 4, 8), (x[0], s, 4, 8), (x, s.cpu(), 4, 8), (x, s[:4], 4, 8),
                 (x[:1].expand(8, 100), s, 4, 8)):
        with pytest.raises(ValueError):
            beam_select(*args)
    with pytest.raises(TypeError):
        beam_select(x.to(torch.bfloat16), s, 4, 8)
    with pytest.raises(ValueError):
        beam_select(x, s, 4, 8, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))


# --------------------------------------------------------------------------------------------------------------- states reordered --
def _moved(t, parents, slot0, first, count):
    out = t.clone()
    beams = parents.shape[1]
    for g, row in enumerate(parents.tolist()):
        for b, p in enumerate(row):
            if 0 <= p < beams:
                d, s = slot0 + g * beams + b, slot0 + g * beams + p
                if count is None:
                    out[d] = t[s]
                else:
                    out[d, :, first:first + count] = t[s, :, first:first + count]
    return out


def _map(kind, groups, beams, rng):
    if kind == "permutation":
        return [rng.sample(range(beams), beams) for _ in range(groups)]
    if kind == "one":
        return [[rng.randrange(beams)] * beams for _ in range(groups)]
    if kind == "same":
        return [list(range(beams)) for _ in range(groups)]
    if kind == "shift":
        return [[(b + 1) % beams for b in range(beams)] for _ in range(groups)]
    return [[rng.randrange(-1, beams + 1) for _ in range(beams)] for _ in range(groups)]


@pytest.mark.parametrize("kind", ["permutation", "one", "same", "shift", "any"])
@pytest.mark.parametrize("beams", [1, 2, 4, 5, 8, 16, 31, 32])
def test_reorder_in_place(kind, beams):
    rng = random.Random(beams)
    parents = torch.tensor(_map(kind, 3, beams, rng), dtype=torch.int32)
    slots = 3 * beams + 2
    bufs = [torch.randn(slots, 3, 20, 24, device="cuda").to(F16), torch.randn(slots, 3, 20, 24, device="cuda").to(F16), torch.randn(slots, 2, 13, 5, device="cuda"),
            torch.randint(0, 100, (slots, 1, 11, 7), device="cuda", dtype=torch.int8)]
    for slot0, first, count in ((0, 0, 20), (2, 3, 8), (1, 10, 1), (0, 5, 0)):
        count = min(count, 11 - first)
        want = [_moved(t, parents, slot0, first, count) for t in bufs]
        reorder_slots(bufs, parents.cuda(), slot0=slot0, first=first, count=count)
        assert all(torch.equal(a, b) for a, b in zip(bufs, want))
    states = [torch.randn(slots, 77, device="cuda"), torch.randn(slots, 4, 4, 16, device="cuda"), torch.arange(slots, device="cuda")]
    want = [_moved(t, parents, 1, 0, None) for t in states]
    reorder_slots(states, parents.cuda(), slot0=1)
    assert all(torch.equal(a, b) for a, b in zip(states, want))


def test_reorder_more_buffers_than_one_launch_takes():
    bufs = [torch.randn(4, 1, 6, 8, device="cuda").to(F16) for _ in range(150)]
    parents = torch.tensor([[1, 0, 3, 3]], dtype=torch.int32)
    want = [_moved(t, parents, 0, 1, 4) for t in bufs]
    reorder_slots(bufs, parents.cuda(), first=1, count=4)
    assert all(torch.equal(a, b) for a, b in zip(bufs, want))


def test_reorder_replayed_in_a_graph():
    t = torch.randn(4, 2, 30, 64, device="cuda").to(F16)
    parents = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        reorder_slots([t], parents, first=2, count=20)
    for row in ([1, 0, 3, 2], [0, 1, 2, 3], [2, 2, 0, 1]):
        parents.copy_(torch.tensor([row], dtype=torch.int32))
        want = _moved(t, parents.cpu(), 0, 2, 20)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(t, want)


def test_reorder_offsets_beyond_32_bits():
    t = torch.zeros(4, 1, 1 << 23, 128, dtype=F16, device="cuda")
    t[3, 0, -2:] = 3.0
    t[2, 0, -2:] = 2.0
    reorder_slots([t], torch.tensor([[3, 1, 3, 2]], dtype=torch.int32, device="cuda"), first=(1 << 23) - 2, count=2)
    assert (t[0, 0, -2:] == 3).all() and (t[2, 0, -2:] == 3).all() and (t[3, 0, -2:] == 2).all() and not t[1].any() and not t[0, 0, :-2].any()


def test_reorder_refusals():
    t = torch.zeros(8, 2, 10, 16, dtype=F16, device="cuda")
    p = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    for args, kw in ((([t, t], p), {}), (([t[:7]], p), {}), (([t], p), dict(slot0=1)), (([t], p), dict(first=3)), (([t], p), dict(first=3, count=8)), (([t], p), dict(count=-1)),
                     (([t.transpose(1, 2)], p), {}), (([t.view(8, -1)], p), dict(count=2)), (([t.cpu()], p), {}), (([t], p.long()), {}), (([t], p.view(-1)), {})):
        with pytest.raises(ValueError):
            reorder_slots(*args, **kw)
    whole = torch.zeros(16, 4, 64, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        reorder_slots([whole, whole[4:]], p)


def test_reorder_refuses_parents_inside_a_buffer():
    t = torch.zeros(4, 2, 16, 64, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        reorder_slots([torch.zeros_like(t), t], t[3, 0, 0, :4].view(1, 4))
    both = torch.zeros(4 * 64 + 4, dtype=torch.int32, device="cuda")                        # (beside it they are fine)
    both[:256] = torch.arange(256)
    both[256:] = torch.tensor([3, 1, 0, 2])
    reorder_slots([both[:256].view(4, 64)], both[256:].view(1, 4))
    assert torch.equal(both[:256].view(4, 64).cpu(), torch.arange(256, dtype=torch.int32).view(4, 64)[[3, 1, 0, 2]])


def test_reorder_refuses_buffers_that_require_gradients():
    t, p = torch.arange(8.0, device="cuda").view(4, 2), torch.tensor([[1, 0, 2, 2]], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="no backward"):
        reorder_slots([t, t.clone().requires_grad_()], p)
    assert torch.equal(t, torch.arange(8.0, device="cuda").view(4, 2))
    with torch.no_grad():
        reorder_slots(iter([t, t.clone().requires_grad_()]), p)
    assert t.tolist() == [[2.0, 3.0], [0.0, 1.0], [4.0, 5.0], [4.0, 5.0]]
