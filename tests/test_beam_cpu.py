"""Beam search's operators: what they refuse, before any launch (CPU)."""
import ctypes

import pytest
import torch

from onebit_amd import _lib
from onebit_amd.beam import _Prefix, beam_select, reorder_slots, shared_prefix_attention, shared_prefix_workspace

E_ARG, E_SHAPE, E_ALIGN, E_DTYPE, E_WSPACE = -1, -2, -3, -4, -5


@pytest.fixture(scope="module")
def buf():
    b = ctypes.create_string_buffer(8192)
    return (ctypes.addressof(b) + 255) & ~255, b


def _attention(a, **kw):
    lib = _lib.load()
    g = kw.get("groups", [(0, 2, 0, 10, 0)])
    arr = (_Prefix * max(len(g), 1))(*[_Prefix(*x) for x in g])
    return lib.onebit_attention_shared_rows(kw.get("q", a), kw.get("pk", a), a, a, a, kw.get("o", a), None, kw.get("arr", arr), len(g), None, kw.get("pos", a),
                                            kw.get("rows", 2), kw.get("H", 4), kw.get("hkv", 2), kw.get("D", 64), kw.get("pslots", 1), kw.get("plen", 10),
                                            kw.get("slots", 2), kw.get("max_len", 16), kw.get("own", 16), kw.get("ws", a), kw.get("nb", 1 << 30), None)


def test_attention_refuses(buf):
    a, _ = buf
    assert _attention(a, D=12) == E_SHAPE and _attention(a, D=136) == E_SHAPE and _attention(a, hkv=3) == E_SHAPE
    assert _attention(a, rows=-1) == E_ARG and _attention(a, slots=0) == E_ARG and _attention(a, own=-1) == E_ARG
    assert _attention(a, rows=0, groups=[]) == 0
    for bad in ([(0, 1, 0, 10, 0)], [(0, 3, 0, 10, 0)], [(1, 2, 0, 10, 0)], [(0, 1, 0, 10, 0), (0, 1, 0, 10, 0)], [(0, 2, 1, 10, 0)], [(0, 2, -1, 10, 0)],
                [(0, 2, 0, 11, 0)], [(0, 2, 0, -1, 0)], [(0, 2, 0, 10, -1)], [(0, 0, 0, 1, 0), (0, 2, 0, 1, 0)], []):
        assert _attention(a, groups=bad) == E_SHAPE, bad
    assert _attention(a, q=None) == E_ARG and _attention(a, pos=None) == E_ARG and _attention(a, pk=None) == E_ARG
    assert _attention(a, q=a + 2) == E_ALIGN and _attention(a, pk=a + 8) == E_ALIGN and _attention(a, o=a + 4) == E_ALIGN
    assert _attention(a, ws=None) == E_WSPACE and _attention(a, nb=8) == E_WSPACE and _attention(a, ws=a + 4) == E_WSPACE
    assert _attention(a, max_len=1 << 31) == E_ARG and _attention(a, rows=70000, groups=[(0, 70000, 0, 10, 0)]) == E_ARG


def test_attention_scratch_grows_with_its_parts():
    f = lambda groups, rows, own: shared_prefix_workspace(groups, rows, 8, 8, 128, own, device="cpu").numel()
    assert f([(0, 4, 0, 5000, 0)], 4, 20) >= 4 * 8 * 2 * 130 * 4
    assert f([(0, 4, 0, 100000, 0)], 4, 20) > f([(0, 4, 0, 5000, 0)], 4, 20)
    with pytest.raises(ValueError, match="rows"):
        f([(0, 4, 0, 100, 0)], 5, 20)
    with pytest.raises(ValueError, match="groups are"):
        f([(0, 4, 0, 100)], 4, 20)


def _select(a, **kw):
    return _lib.load().onebit_beam_select(kw.get("x", a), kw.get("ld", 100), kw.get("dt", 0), a, kw.get("groups", 2), kw.get("beams", 4), kw.get("vocab", 100),
                                          kw.get("keep", 8), kw.get("out", a), a, a, kw.get("ws", a), kw.get("nb", 1 << 30), None)


def test_select_refuses(buf):
    a, _ = buf
    assert _select(a, groups=-1) == E_ARG and _select(a, vocab=0) == E_ARG and _select(a, groups=0) == 0
    assert _select(a, beams=0) == E_SHAPE and _select(a, beams=33) == E_SHAPE and _select(a, keep=0) == E_SHAPE and _select(a, keep=65) == E_SHAPE
    assert _select(a, vocab=1 << 21, ld=1 << 21) == E_ARG and _select(a, groups=20000) == E_ARG and _select(a, groups=1 << 62) == E_ARG
    assert _select(a, dt=2) == E_DTYPE and _select(a, ld=99) == E_SHAPE and _select(a, x=None) == E_ARG and _select(a, out=None) == E_ARG
    assert _select(a, x=a + 1) == E_ALIGN and _select(a, out=a + 2) == E_ALIGN
    assert _select(a, ws=None) == E_WSPACE and _select(a, nb=64) == E_WSPACE


def _reorder(a, **kw):
    ptrs = (ctypes.c_void_p * 2)(a, kw.get("second", a + 4096))
    return _lib.load().onebit_reorder_slots(ptrs, kw.get("n", 2), kw.get("parents", a), kw.get("groups", 1), kw.get("beams", 4), kw.get("slot", 256), kw.get("outer", 2),
                                            kw.get("row", 128), kw.get("first", 0), kw.get("nb", 128), None)


def test_reorder_refuses(buf):
    a, _ = buf
    assert _reorder(a, n=-1) == E_ARG and _reorder(a, first=-1) == E_ARG and _reorder(a, nb=-1) == E_ARG and _reorder(a, parents=None) == E_ARG
    assert _reorder(a, second=None) == E_ARG and _reorder(a, parents=a + 1) == E_ALIGN
    assert _reorder(a, beams=0) == E_SHAPE and _reorder(a, beams=33) == E_SHAPE and _reorder(a, groups=65536) == E_SHAPE
    assert _reorder(a, first=16) == E_SHAPE and _reorder(a, slot=255) == E_SHAPE and _reorder(a, outer=3) == E_SHAPE
    assert _reorder(a, outer=1 << 60) == E_SHAPE and _reorder(a, slot=1 << 60) == E_SHAPE
    for nothing in (dict(n=0), dict(groups=0), dict(nb=0), dict(outer=0)):
        assert _reorder(a, **nothing) == 0, nothing


def test_python_checks_name_the_mistake():
    q, c = torch.zeros(2, 4, 64, dtype=torch.float16), torch.zeros(2, 4, 16, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        shared_prefix_attention(q, None, None, c, c, [(0, 2, 0, 0, 0)], None, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        beam_select(torch.zeros(4, 10), torch.zeros(4), 4, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        reorder_slots([c], torch.zeros(1, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="parents"):
        reorder_slots([c], torch.zeros(1, 2))


def test_shared_step_refuses(buf):
    from onebit_amd.engine import _Layer, _MixedState, _Model
    a, _ = buf
    lib = _lib.load()
    m = _Model(1, 128, 352, 2, 2, 64, 96, 32, 1e-6, 1e-5, (_Layer * 1)(), a, a, a, a, a)
    st = _MixedState(ctypes.sizeof(_MixedState), 2, 2, 0, 1, 4, 0, 0, a, a, a, None, a, a, None, a, a, a, 1 << 30)

    def call(groups, own=8, ws=a, nb=1 << 20):
        arr = (_Prefix * max(len(groups), 1))(*[_Prefix(*g) for g in groups])
        return lib.onebit_mixed_step_shared(ctypes.byref(m), ctypes.byref(st), arr, len(groups), own, ws, nb, None)
    assert call([(0, 2, 4, 10, 10)]) == E_SHAPE and b"prefix" in lib.onebit_last_error()           # slot 4 of 4
    assert call([(0, 2, 0, 33, 33)]) == E_SHAPE and call([(0, 1, 0, 10, 10)]) == E_SHAPE and call([]) == E_SHAPE
    assert call([(0, 2, 0, 10, 10)], ws=None) == E_WSPACE and call([(0, 2, 0, 10, 10)], nb=1) == E_WSPACE
    assert lib.onebit_mixed_step_shared(None, ctypes.byref(st), None, 0, 0, None, 0, None) == E_ARG
    st.struct_size = 8
    assert call([(0, 2, 0, 10, 10)]) == E_ARG and b"struct_size" in lib.onebit_last_error()


class _Slots:
    """A search's bookkeeping alone: candidates in, slots out."""

    def __init__(self, beams, penalty=1.0, early=False):
        from onebit_amd.search import _Prompt
        self.p = _Prompt(beams, penalty, early)


def test_hypotheses_keep_their_slots():
    p = _Slots(3).p
    p.take([(-1.0, 0, 5), (-2.0, 0, 6), (-3.0, 0, 7), (-4.0, 0, 8)], None)
    assert [(t, s) for _, t, s in p.live] == [([5], 0), ([6], 1), ([7], 2)]
    # the second goes on twice, the first not at all: its slot takes the second's state
    assert p.take([(-2.5, 1, 1), (-3.5, 2, 2), (-3.6, 1, 3)], None) == [1, 1, 2]
    assert [(t, s) for _, t, s in p.live] == [([6, 1], 1), ([7, 2], 2), ([6, 3], 0)]
    # a beam is a rank, not a slot
    assert p.take([(-4.0, 2, 0), (-4.1, 2, 1), (-4.2, 2, 2)], None) == [0, 0, 0]
    assert [s for _, _, s in p.live] == [0, 1, 2]


def test_finished_hypotheses():
    p = _Slots(2).p
    p.take([(-1.0, 0, 9), (-1.5, 0, 4), (-1.6, 0, 5), (-9.0, 0, 6)], {9})
    assert p.finished == [(-1.0, [9])] and [t for _, t, _ in p.live] == [[4], [5]] and not p.done
    p.take([(-1.7, 1, 4), (-1.8, 0, 4), (-1.9, 0, 9)], {9})
    assert len(p.finished) == 1                                        # an end behind all that could go on is none
    p.take([(-2.0, 0, 9), (-2.1, 1, 4), (-2.2, 1, 5)], {9})
    assert [t for _, t in p.finished] == [[5, 4, 9], [9]] and not p.done       # -2/3, -1; live ones at -0.7
    p.take([(-7.0, 0, 4), (-7.5, 1, 5)], {9})
    assert p.done and p.results() == p.finished
    early = _Slots(1, early=True).p
    early.take([(-5.0, 0, 9), (-5.1, 0, 4)], {9})
    assert early.done
    empty = _Slots(2).p
    empty.take([(float("-inf"), -1, -1)] * 4, None)
    assert empty.done and empty.results() == []


class _NoEngine:
    """A search's engine that must not be asked for anything."""
    batch, beams, max_len, vocab, device = 1, 32, 100, 50, "cpu"

    def prime(self, prompts):
        raise AssertionError("nothing to prime")


def test_search_refuses_more_candidates_than_are_kept():
    from onebit_amd.search import beam_search
    with pytest.raises(ValueError, match="96 candidates"):
        beam_search(_NoEngine(), [[1, 2]], 5, eos={3, 4})


def test_search_of_no_token():
    from onebit_amd.search import beam_search
    assert beam_search(_NoEngine(), [[1, 2]], 0) == [[(0.0, [])]]


def test_groups_beyond_32_bits():
    with pytest.raises(ValueError, match="32 bits"):
        shared_prefix_workspace([(0, 2, 0, 1 << 32, 0)], 2, 4, 4, 64, 10, "cpu")
    with pytest.raises(ValueError, match="32 bits"):
        shared_prefix_workspace([(0, 2, -(1 << 40), 3, 0)], 2, 4, 4, 64, 10, "cpu")


def test_command_line_refuses_a_search_s_options_without_one(capsys):
    from onebit_amd.cli import main
    for extra in (["--eos", "3"], ["--length-penalty", "2"]):
        with pytest.raises(SystemExit):
            main(["generate", "--model", "none", "--prompt", "1", *extra])
        assert "--num-beams" in capsys.readouterr().err


def _pieces():
    """Addresses in one allocation, 1 MiB apart (never launched on: every call below is refused)."""
    b = ctypes.create_string_buffer(17 << 20)
    a = (ctypes.addressof(b) + 255) & ~255
    return b, [a + (i << 20) for i in range(16)]


def test_attention_refuses_overlaps():
    """q, o [2, 4, 64] 1024 bytes, own caches [2, 2, 16, 64] 8192, prefix caches [1, 2, 10, 64] 2560, row indices 8: one byte into any of them, from either end."""
    keep, p = _pieces()
    lib = _lib.load()
    arr = (_Prefix * 1)(_Prefix(0, 2, 0, 10, 0))
    size = dict(q=1024, pk=2560, pv=2560, k=8192, v=8192, o=1024, h=512, slot=8, pos=8)
    size["ws"] = lib.onebit_attention_shared_scratch_bytes(arr, 1, 2, 4, 2, 64, 16)
    at = dict(zip(size, p))

    def call(**kw):
        w = {**at, **kw}
        return lib.onebit_attention_shared_rows(w["q"], w["pk"], w["pv"], w["k"], w["v"], w["o"], w["h"], arr, 1, w["slot"], w["pos"], 2, 4, 2, 64, 1, 10, 2, 16, 16,
                                                w["ws"], size["ws"], None)
    for written in ("o", "ws"):
        step = 8 if written == "o" else 16
        for other in size:
            if other == written:
                continue
            for where in (at[other], at[other] - size[written] + step, at[other] + (size[other] - 1) // step * step):
                assert call(**{written: where}) == E_ARG and b"overlap" in lib.onebit_last_error(), (written, other, where - at[other])


def test_attention_refuses_too_many_workgroups_before_the_first_launch():
    """64 groups of a row, which one launch takes, then 65471 rows of 512 key heads, 2^25 workgroups."""
    lib = _lib.load()
    groups = [(r, 1, 0, 0, 0) for r in range(64)] + [(64, 65471, 0, 0, 0)]
    arr = (_Prefix * 65)(*[_Prefix(*g) for g in groups])
    at = [(i + 1) << 40 for i in range(6)]
    rc = lib.onebit_attention_shared_rows(at[0], None, None, at[1], at[2], at[3], None, arr, 65, None, at[4], 65535, 512, 512, 8, 0, 0, 65535, 16, 16, at[5], 1 << 39, None)
    assert rc == E_ARG and b"too many workgroups" in lib.onebit_last_error()


def test_reorder_refuses_parents_inside_a_buffer():
    """Two buffers of 4 slots of 256 bytes, parents of 16 bytes: at either end of either buffer."""
    keep, p = _pieces()
    lib = _lib.load()
    for first in (0, 1):
        bufs = (ctypes.c_void_p * 2)(p[first], p[1 - first])
        for at in (p[0] - 12, p[0], p[0] + 1020):
            assert lib.onebit_reorder_slots(bufs, 2, at, 1, 4, 256, 2, 128, 0, 128, None) == E_ARG and b"overlap" in lib.onebit_last_error()


def test_select_refuses_overlaps():
    """2 groups of 4 rows of 100 fp32 logits (pitch 128: 3984 bytes), 8 kept: one entry into any other piece of memory, from either end."""
    keep, p = _pieces()
    lib = _lib.load()
    size = dict(out=64, beam=64, token=64, ws=lib.onebit_beam_select_scratch_bytes(8, 100, 8), scores=32, x=(7 * 128 + 100) * 4)
    at = dict(zip(size, p))

    def call(**kw):
        w = {**at, **kw}
        return lib.onebit_beam_select(w["x"], 128, 1, w["scores"], 2, 4, 100, 8, w["out"], w["beam"], w["token"], w["ws"], size["ws"], None)
    for written in ("out", "beam", "token", "ws"):
        step = 16 if written == "ws" else 4
        for other in size:
            if other == written:
                continue
            for where in (at[other], at[other] - size[written] + step, at[other] + (size[other] - 1) // step * step):
                assert call(**{written: where // step * step}) == E_ARG and b"overlap" in lib.onebit_last_error(), (written, other, where - at[other])


def test_tensors_that_require_gradients_are_refused():
    half = lambda *s: torch.zeros(*s, dtype=torch.float16)
    pos, groups = torch.zeros(2, dtype=torch.int32), [(0, 2, 0, 4, 0)]
    for i in range(6):
        t = [half(2, 4, 64), half(1, 4, 4, 64), half(1, 4, 4, 64), half(2, 4, 16, 64), half(2, 4, 16, 64), half(256)]
        t[i].requires_grad_()
        call = lambda: shared_prefix_attention(t[0], t[1], t[2], t[3], t[4], groups, None, pos, h_next=t[5])
        with pytest.raises(ValueError, match="no backward"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):                    # (refused for the next reason only)
            call()
    for i in range(2):
        t = [torch.zeros(4, 10), torch.zeros(4)]
        t[i].requires_grad_()
        with pytest.raises(ValueError, match="no backward"):
            beam_select(t[0], t[1], 4, 8)


def test_what_a_search_refuses_takes_no_memory(monkeypatch):
    """More end tokens than candidates are kept, a prompt of no token: no engine is built, and none is kept."""
    from onebit_amd import search

    def build(*args):
        raise AssertionError("an engine for a search that is refused")
    monkeypatch.setattr(search, "LlamaBeams", build)
    engines = {}
    for prompts, beams, eos in (([[1, 2]], 32, {3, 4}), ([[1], []], 2, None), ([], 2, None)):
        with pytest.raises(ValueError):
            search.beam_rows(object(), prompts, 5, 100, engines, beams, eos)
    assert not engines


def test_slots_of_one_search_at_a_time(monkeypatch):
    """An engine that is kept serves the next search of its sizes; one for other sizes takes its place, next to what greedy generation keeps."""
    from onebit_amd import search
    built, engines, greedy = [], {(2, 256): "greedy"}, {(2, 256)}

    class Engine:
        def __init__(self, model, batch, beams, max_len):
            assert set(engines) == greedy                            # (the old one's memory is free before the new one's is taken)
            built.append((batch, beams, max_len))
    monkeypatch.setattr(search, "LlamaBeams", Engine)
    monkeypatch.setattr(search, "beam_search", lambda eng, prompts, *a: [[(0.0, [1])] for _ in prompts])
    for prompts, new in (([[1]], 5), ([[1]], 9), ([[1]], 300), ([[1], [2]], 300), ([[1]], 5)):
        search.beam_rows(object(), prompts, new, 1000, engines, 4)
        assert len(engines) == 2
    assert built == [(1, 4, 256), (1, 4, 512), (2, 4, 512), (1, 4, 256)]


def test_command_line_searches_max_batch_prompts_at_a_time(monkeypatch, capsys):
    import types

    import onebit_amd.registry as registry
    import onebit_amd.search as search
    from onebit_amd.cli import main
    calls = []

    def rows(model, prompts, new, limit, engines, beams, eos, penalty):
        calls.append((prompts, id(engines)))
        return [[p[0] + 100] for p in prompts]
    monkeypatch.setattr(search, "beam_rows", rows)
    monkeypatch.setattr(registry, "load_model", lambda *a, **kw: None)
    monkeypatch.setattr(registry, "find_family", lambda path: types.SimpleNamespace(max_positions=lambda model: 64))
    argv = ["generate", "--model", "none", "--num-beams", "3"] + [x for i in range(5) for x in ("--prompt", str(i))]
    assert main(argv + ["--max-batch", "2"]) == 0
    assert [p for p, _ in calls] == [[[0], [1]], [[2], [3]], [[4]]] and len({e for _, e in calls}) == 1
    assert capsys.readouterr().out.splitlines() == [f'{{"request": {i}, "tokens": [{100 + i}]}}' for i in range(5)]
    calls.clear()
    assert main(argv) == 0 and len(calls) == 1
    with pytest.raises(SystemExit):
        main(argv + ["--prefill-chunk", "8"])
    assert "--prefill-chunk" in capsys.readouterr().err
