"""Beam search's operators on the native library (include/onebit.h): attention of hypotheses that share their prompt, the choice of the next
hypotheses from their logits, and their states brought to the slots that go on with them.

All three enqueue on the current stream of their tensors' device and never synchronise; they can be captured into a HIP graph (host
arguments -- the groups, lengths, positions -- are fixed by the capture, device tensors are read by every replay).  Results carry no
gradients; tensors that require them are refused unless gradients are off.  A workspace may be kept
between calls; calls that may run at the same time (other streams, graphs replayed next to each other) need one each.  There is no CPU fallback."""
from __future__ import annotations

import ctypes
import struct
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from .bitnet import _dtype_code, _raw_stream as _raw, _require_gpu, _stream_ptr

MAX_BEAMS, MAX_KEEP = 32, 64


class _Prefix(ctypes.Structure):          # onebit_prefix_t
    _fields_ = [("row0", ctypes.c_int32), ("n", ctypes.c_int32), ("slot", ctypes.c_int32), ("len", ctypes.c_int32), ("first", ctypes.c_int32)]


_GROUP = struct.Struct("5i")          # onebit_prefix_t


def _prefixes(groups) -> bytes:
    """The groups as an array of onebit_prefix_t."""
    try:
        return _GROUP.pack(*groups[0]) if len(groups) == 1 else b"".join([_GROUP.pack(*g) for g in groups])
    except struct.error as e:
        raise ValueError(f"groups are (first row, rows, prefix slot, prefix length, first own position) each, whole numbers of 32 bits, not {list(groups)!r}") from e


def _call(name: str, index: int, *args):
    """The library's function on the current stream of device ``index``."""
    lib = _lib._lib or _lib.load()
    if index == _get_device():
        rc = getattr(lib, name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = getattr(lib, name)(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


_grad = torch.is_grad_enabled
_get_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = _raw if _raw is not None else lambda index: _stream_ptr(torch.device("cuda", index))
_F16, _F32, _I32, _U8 = torch.float16, torch.float32, torch.int32, torch.uint8


def _on(index: int, what: str, *tensors):
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError(f"{what}: tensors on cuda:{index} and {t.device}")


def _no_gradient(what: str):
    raise ValueError(f"{what}: serves only, there is no backward pass: call it under torch.no_grad(), or with tensors that do not require gradients")


def _check_rows(what: str, rows: int, **tensors):
    for name, t in tensors.items():
        if t is not None and not (t.dtype is _I32 and t.shape == (rows,) and t.is_contiguous()):
            raise ValueError(f"{what}: {name} must be a contiguous int32 tensor of {rows} entries")


def shared_prefix_workspace(groups: Sequence[Tuple[int, int, int, int, int]], rows: int, heads: int, kv_heads: int, head_dim: int, max_own: int,
                            device="cuda") -> torch.Tensor:
    """Scratch memory for ``shared_prefix_attention`` calls of these groups and sizes, and of any that need no more: zero-filled once, every call leaves
    its counters at zero."""
    lib = _lib.load()
    n = lib.onebit_attention_shared_scratch_bytes(_prefixes(groups), len(groups), rows, heads, kv_heads, head_dim, max_own)
    if rows > 0 and n == 0:
        raise ValueError(f"shared_prefix_workspace: {lib.onebit_last_error().decode('utf-8', 'replace')}")
    return torch.zeros(max(int(n), 1), dtype=torch.uint8, device=device)


def shared_prefix_attention(q: torch.Tensor, prefix_k: Optional[torch.Tensor], prefix_v: Optional[torch.Tensor], k_cache: torch.Tensor, v_cache: torch.Tensor,
                            groups: Sequence[Tuple[int, int, int, int, int]], row_slot: Optional[torch.Tensor], row_pos: torch.Tensor,
                            max_own: Optional[int] = None, h_next: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                            workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of single-token rows over a prefix that they share and positions of their own (``onebit_attention_shared_rows``).

    ``q`` [rows, heads, D] fp16 (D a multiple of 8, at most 128).  ``groups``: ``(first row, rows, slot, length, first)`` each, tiling the rows
    in order; a group's rows attend to positions 0 .. length - 1 of ``slot`` in ``prefix_k`` / ``prefix_v`` [prefix slots, kv heads, prefix positions, D],
    and row r to positions first .. row_pos[r] of slot ``row_slot[r]`` (None: slot r) in ``k_cache`` / ``v_cache`` [slots, kv heads, positions, D].  The two
    pairs may be the same tensors; without any prefix the first may be None.  ``row_slot`` / ``row_pos``: int32 on the device; a row whose slot
    or position lies outside is idle and keeps what ``out`` holds (zeros without ``out``).  ``out`` overlaps no input.  ``max_own``: bound on the rows' own positions, those
    beyond it are not attended (None: all that fit the cache).  ``h_next`` [heads * D]: the result times this."""
    what = "shared_prefix_attention"
    if _grad() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad or (prefix_k is not None and prefix_k.requires_grad) or
                    (prefix_v is not None and prefix_v.requires_grad) or (h_next is not None and h_next.requires_grad) or (out is not None and out.requires_grad)):
        _no_gradient(what)
    _require_gpu(q, what)
    shape = q.shape
    if len(shape) != 3 or q.dtype is not _F16 or not q.is_contiguous():
        raise ValueError(f"{what}: q must be a contiguous float16 [rows, heads, D]")
    rows, heads, dim = shape
    own = k_cache.shape
    if not (len(own) == 4 and own[3] == dim and v_cache.shape == own and k_cache.dtype is _F16 and v_cache.dtype is _F16 and k_cache.is_contiguous() and
            v_cache.is_contiguous()):
        raise ValueError(f"{what}: own caches must be contiguous float16 [slots, kv heads, positions, {dim}], not {tuple(own)} / {tuple(v_cache.shape)}")
    slots, kv_heads, max_len, _ = own
    index = q.get_device()
    p_slots = p_len = p_k = p_v = 0
    if prefix_k is not None and prefix_v is not None:
        pre = prefix_k.shape
        if not (len(pre) == 4 and pre[3] == dim and pre[1] == kv_heads and prefix_v.shape == pre and prefix_k.dtype is _F16 and prefix_v.dtype is _F16 and
                prefix_k.is_contiguous() and prefix_v.is_contiguous() and prefix_k.get_device() == index and prefix_v.get_device() == index):
            raise ValueError(f"{what}: prefix caches must be contiguous float16 [slots, {kv_heads}, positions, {dim}] on {q.device}, not {tuple(pre)} / "
                             f"{tuple(prefix_v.shape)} on {prefix_k.device}")
        p_slots, _, p_len, _ = pre
        p_k, p_v = prefix_k.data_ptr(), prefix_v.data_ptr()
    elif prefix_k is not None or prefix_v is not None:
        raise ValueError(f"{what}: prefix keys without values, or values without keys")
    if row_pos is None:
        raise ValueError(f"{what}: row_pos is needed")
    if not (row_pos.dtype is _I32 and row_pos.dim() == 1 and row_pos.numel() == rows and row_pos.is_contiguous()):
        _check_rows(what, rows, row_pos=row_pos)
    slot, scale, where = None, None, index
    if row_slot is not None:
        if not (row_slot.dtype is _I32 and row_slot.dim() == 1 and row_slot.numel() == rows and row_slot.is_contiguous()):
            _check_rows(what, rows, row_slot=row_slot)
        slot, where = row_slot.data_ptr(), row_slot.get_device()
    if h_next is not None:
        if h_next.dtype is not _F16 or h_next.numel() != heads * dim or not h_next.is_contiguous():
            raise ValueError(f"{what}: h_next must be contiguous float16 of {heads * dim} entries")
        scale = h_next.data_ptr()
        where = where if h_next.get_device() == index else -1
    if out is None:
        out = torch.zeros_like(q)
    elif out.shape != shape or out.dtype is not _F16 or not out.is_contiguous() or out.data_ptr() == q.data_ptr() != 0:
        raise ValueError(f"{what}: out must be like q and not q")
    arr = _prefixes(groups)
    if max_own is None:
        max_own = max([0] + [max_len - int(g[4]) for g in groups])
    if workspace is None:
        workspace = shared_prefix_workspace(groups, rows, heads, kv_heads, dim, max_own, q.device)
    elif workspace.dtype is not _U8 or not workspace.is_contiguous():
        raise ValueError(f"{what}: the workspace must be contiguous uint8")
    if not (k_cache.get_device() == index == v_cache.get_device() == row_pos.get_device() == out.get_device() == workspace.get_device()) or where != index:
        _on(index, what, k_cache, v_cache, row_slot, row_pos, h_next, out, workspace)
    _call("onebit_attention_shared_rows", index, q.data_ptr(), p_k, p_v, k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), scale, arr, len(groups),
          slot, row_pos.data_ptr(), rows, heads, kv_heads, dim, p_slots, p_len, slots, max_len, max_own, workspace.data_ptr(), workspace.numel())
    return out


def beam_select_workspace(rows: int, vocab: int, keep: int, device="cuda") -> torch.Tensor:
    """Scratch memory for ``beam_select`` calls of these sizes and smaller ones: zero-filled once, every call leaves its counters at zero."""
    return torch.zeros(max(int(_lib.load().onebit_beam_select_scratch_bytes(rows, vocab, keep)), 1), dtype=torch.uint8, device=device)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, beams: int, keep: int,
                workspace: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``keep`` best continuations of every group of ``beams`` hypotheses (``onebit_beam_select``): ``logits`` [groups * beams, vocab] float16 or
    float32 (rows may be strided), ``scores`` float32 [groups * beams], the hypotheses' sums of log probabilities.  Returns scores (float32), beams and
    tokens (int32), [groups, keep] each, best first: views of one int32 tensor [3, groups, keep].  Values are added and compared in 64 bits, equal ones by
    beam, logit, token; a row's log-sum in them is off by some 1e-7 (bound: ``onebit_beam_select``), which is how far the order between rows is exact.  A continuation of probability zero is none: places that remain hold -inf, -1, -1."""
    values, beam, token = select_packed(logits, scores, beams, keep, workspace).unbind(0)
    return values.view(_F32), beam, token


def select_packed(logits: torch.Tensor, scores: torch.Tensor, beams: int, keep: int, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``beam_select``'s int32 tensor [3, groups, keep] as one: the scores' bits, beams, tokens."""
    if _grad() and (logits.requires_grad or scores.requires_grad):
        _no_gradient("beam_select")
    _require_gpu(logits, "beam_select")
    shape = logits.shape
    if len(shape) != 2 or (shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("beam_select: logits must be [rows, vocab] with adjacent columns")
    rows, vocab = shape
    if not 1 <= beams <= MAX_BEAMS or rows % beams:
        raise ValueError(f"beam_select: {rows} rows in groups of {beams} hypotheses (1 .. {MAX_BEAMS})")
    if not 1 <= keep <= MAX_KEEP:
        raise ValueError(f"beam_select: {keep} kept (1 .. {MAX_KEEP})")
    if scores.dtype is not _F32 or scores.numel() != rows or not scores.is_contiguous():
        raise ValueError(f"beam_select: scores must be contiguous float32 of {rows} entries")
    if workspace is None:
        workspace = beam_select_workspace(rows, vocab, keep, logits.device)
    elif workspace.dtype is not _U8 or not workspace.is_contiguous():
        raise ValueError("beam_select: the workspace must be contiguous uint8")
    index = logits.get_device()
    if not scores.get_device() == index == workspace.get_device():
        _on(index, "beam_select", scores, workspace)
    groups = rows // beams
    packed = torch.empty_strided((3, groups, keep), (groups * keep, keep, 1), dtype=_I32, device=logits.device)
    p, ld = packed.data_ptr(), logits.stride(0)
    if rows == 1:
        ld = max(ld, vocab)
    _call("onebit_beam_select", index, logits.data_ptr(), ld, _dtype_code(logits.dtype), scores.data_ptr(), groups, beams, vocab, keep, p,
          p + 4 * groups * keep, p + 8 * groups * keep, workspace.data_ptr(), workspace.numel())
    return packed


def reorder_slots(buffers: Sequence[torch.Tensor], parents: torch.Tensor, slot0: int = 0, first: int = 0, count: Optional[int] = None) -> None:
    """In every buffer [slots, ...], slot ``slot0 + g * beams + b`` takes what slot ``slot0 + g * beams + parents[g, b]`` held, in place and for any map
    (``onebit_reorder_slots``); ``parents`` int32 [groups, beams] on the device, an entry outside 0 .. beams - 1 leaves its slot as it is.  With ``count``,
    buffers are caches [slots, heads, positions, D] of which positions ``first`` .. ``first + count - 1`` move.  Any dtype; buffers overlap neither each other nor ``parents``."""
    if parents.dim() != 2 or parents.dtype is not _I32 or not parents.is_contiguous():
        raise ValueError("reorder_slots: parents must be a contiguous int32 [groups, beams]")
    _require_gpu(parents, "reorder_slots")
    groups, beams = parents.shape
    if not 1 <= beams <= MAX_BEAMS:
        raise ValueError(f"reorder_slots: {beams} beams (1 .. {MAX_BEAMS})")
    if count is None and first:
        raise ValueError("reorder_slots: first without count")
    if slot0 < 0 or first < 0 or (count is not None and count < 0):
        raise ValueError("reorder_slots: negative slot0, first or count")
    index, slots = parents.get_device(), slot0 + groups * beams
    shapes: dict = {}
    shape = dtype = into = None
    grad = _grad()
    for t in buffers:
        if grad and t.requires_grad:
            _no_gradient("reorder_slots")
        if not t.is_contiguous() or t.get_device() != index:
            raise ValueError(f"reorder_slots: a buffer {tuple(t.shape)} on {t.device} must be contiguous and on {parents.device}")
        if t.shape != shape or t.dtype != dtype:
            shape, dtype = t.shape, t.dtype
            if t.dim() < 1 or shape[0] < slots:
                raise ValueError(f"reorder_slots: a buffer {tuple(shape)} must have {slots} slots")
            size = t.element_size()
            slot = t.stride(0) * size if t.numel() else 0
            if count is None:
                geometry = (slot, 1, slot, 0, slot)
            elif len(shape) != 4 or first + count > shape[2]:
                raise ValueError(f"reorder_slots: positions {first} .. {first + count - 1} of a cache {tuple(shape)}")
            else:
                row = shape[3] * size
                geometry = (slot, shape[1], shape[2] * row, first * row, count * row)
            into = shapes.setdefault((shape[0] * slot, geometry), [])
        into.append(t.data_ptr())
    if groups == 0:
        return
    ends = sorted((p, p + n) for (n, _), ptrs in shapes.items() if n for p in ptrs)
    if any(a[1] > b[0] for a, b in zip(ends, ends[1:])):
        raise ValueError("reorder_slots: buffers overlap")
    for (n, geometry), ptrs in shapes.items():
        if n:
            arr = (ctypes.c_void_p * len(ptrs))(*([p + slot0 * geometry[0] for p in ptrs] if slot0 else ptrs))
            _call("onebit_reorder_slots", index, arr, len(ptrs), parents.data_ptr(), groups, beams, *geometry)
