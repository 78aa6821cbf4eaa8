"""The 8-bit paged cache of attention layers: rows appended to it, its pages read back, attention over it (kernels/pages8.cu, attn_pages8.cu).

Keys and values stand in pages of 64 positions, [page, KV head, position, column], as E4M3 numbers (:class:`Pages8`).  Each page has a unit for each KV head, a power
of two between 2^-15 and 2^7; a value is its number times the unit, and always an f16 number too.  The unit is the least with which the largest magnitude that was
appended to the page fits; larger magnitudes than 57344 become that.  Where an appended row makes the unit grow, the page's other rows are rounded to the new one, and a
row at a page's first position begins the page anew.  Rows have 64 or 128 columns; heads of fewer leave zeros behind theirs.

Tables of pages are [slots, pages] int32: entry i of a slot is the page of its positions 64 i .. 64 i + 63.  Rows whose position is negative hold no token: nothing is
appended for them and their results are left as they are.  So are rows whose slot, position or page is not there.  All calls run on the current stream of the
tensors' device.
"""
from __future__ import annotations

import ctypes as C
import functools
from dataclasses import dataclass

import torch

from .cuda import _check, lib, ptr
from .rows import NO_DIFF, NO_GATE, DiffHeads, F, HeadGate, I, P, _st

PAGE = 64

_Pages8 = _st("_Pages8", [("k", P), ("ku", P), ("v", P), ("vu", P), ("n_pages", I), ("kv_heads", I), ("hd", I)])
_PageTable = _st("_PageTable", [("table", P), ("n_slots", I), ("max_pages", I)])
Append8Args = _st("Append8Args", [("qkv", P), ("ldq", I), ("rows", I), ("n_heads", I), ("dim", I), ("vdim", I), ("q_norm", P), ("k_norm", P), ("eps", F), ("freqs", P),
                                  ("n_rot", I), ("positions", P), ("slots", P), ("segs", P), ("n_segs", I), ("per", I), ("t", _PageTable), ("q_out", P), ("c", _Pages8),
                                  ("head_norm", I), ("v_off", I), ("mscale", F), ("maps", I), ("no_append", I)])
Attn8Args = _st("Attn8Args", [("q", P), ("rows", I), ("n_heads", I), ("vdim", I), ("c", _Pages8), ("t", _PageTable), ("positions", P), ("slots", P), ("segs", P), ("n_segs", I),
                              ("chunk", I), ("window", I), ("keep", I), ("scale", F), ("softcap", F), ("n_splits", I), ("part_acc", P), ("part_ml", P), ("out", P), ("ldo", I),
                              ("out16", I), ("gate", HeadGate), ("diff", DiffHeads)])


@dataclass
class Pages8:
    """Keys or values of a layer: ``codes`` [pages, KV heads, 64, 64 or 128] uint8, ``unit`` [pages, KV heads] fp32."""

    codes: torch.Tensor
    unit: torch.Tensor

    def __post_init__(self):
        c, u = self.codes, self.unit
        if c.dim() != 4 or c.shape[2] != PAGE or c.shape[3] not in (64, 128) or c.dtype != torch.uint8 or not c.is_contiguous():
            raise ValueError(f"Pages8: codes {tuple(c.shape)} {c.dtype}")
        if u.shape != c.shape[:2] or u.dtype != torch.float32 or not u.is_contiguous() or u.device != c.device:
            raise ValueError(f"Pages8: units {tuple(u.shape)} {u.dtype} on {u.device}")

    @classmethod
    def empty(cls, n_pages: int, kv_heads: int, dim: int, device="cuda") -> "Pages8":
        """Pages of zeros for heads of up to ``dim`` columns."""
        if not 1 <= dim <= 128:
            raise ValueError(f"Pages8: heads of {dim} columns")
        return cls(torch.zeros(n_pages, kv_heads, PAGE, 64 if dim <= 64 else 128, device=device, dtype=torch.uint8), torch.ones(n_pages, kv_heads, device=device))

    @property
    def numbers(self) -> torch.Tensor:
        """The codes as E4M3 numbers."""
        return self.codes.view(torch.float8_e4m3fn)


@dataclass
class Portions8:
    """Portions of prompts in a step, of different slots: what :func:`append8` and :func:`attn_prompt8` have to know of them."""

    segs: torch.Tensor               # [n, 4]: first row, rows, slot, position of the first row
    rows: int                        # of all portions
    per: int                         # most pages that a portion's rows go to


def portions8(parts, table: torch.Tensor, *, window: int = 0, keep: int = 0, chunk: int = 0) -> Portions8:
    """``parts``: (first row, rows, slot, position of the first row) of each portion, rows one after the other; the masks are those of the attention."""
    n_slots, max_pages = table.shape
    at, slots = 0, set()
    for row, n, slot, pos in parts:
        if n < 1 or row != at or not 0 <= slot < n_slots or pos < 0 or pos + n > max_pages * PAGE:
            raise ValueError(f"portions8: {n} rows from {row} on at position {pos} of slot {slot}, in a table {tuple(table.shape)}")
        if slot in slots:
            raise ValueError(f"portions8: two portions of slot {slot}")
        at += n
        slots.add(slot)
    if not at:
        raise ValueError("portions8: no rows")
    segs = torch.tensor(parts, dtype=torch.int32).to(table.device)
    return Portions8(segs, at, max((p + n - 1) // PAGE - p // PAGE + 1 for _, n, _, p in parts))


def _on_device(f):
    """Run ``f`` with its first tensor's device current."""
    @functools.wraps(f)
    def call(x, *a, **kw):
        if x.device.type != "cuda":
            raise ValueError(f"{f.__name__}: tensors on {x.device}")
        if x.device.index == torch.cuda.current_device():
            return f(x, *a, **kw)
        with torch.cuda.device(x.device):
            return f(x, *a, **kw)
    return call


def _stream(x: torch.Tensor) -> C.c_void_p:
    return C.c_void_p(torch.cuda.current_stream(x.device).cuda_stream)


def _need(what: str, name: str, t: torch.Tensor | None, dtype, device, *shape, contiguous: bool = True) -> None:
    """A tensor of the type, on the device, of the shape (None: any size) with rows that are one piece."""
    if t is None or t.dtype not in (dtype if isinstance(dtype, tuple) else (dtype,)) or t.device != device or t.dim() != len(shape) or \
            any(s is not None and s != n for s, n in zip(shape, t.shape)) or (not t.is_contiguous() if contiguous else t.numel() and t.stride(-1) != 1):
        raise ValueError(f"{what}: {name} " + ("is missing" if t is None else f"{tuple(t.shape)} {t.dtype} on {t.device}, strides {t.stride()}"))


def _cache(what: str, k: Pages8, v: Pages8, table: torch.Tensor, device) -> tuple:
    if k.codes.shape != v.codes.shape or k.codes.device != device or v.codes.device != device:
        raise ValueError(f"{what}: keys {tuple(k.codes.shape)} on {k.codes.device}, values {tuple(v.codes.shape)} on {v.codes.device}")
    _need(what, "table", table, torch.int32, device, None, None)
    n, g, _, hd = k.codes.shape
    return _Pages8(ptr(k.codes), ptr(k.unit), ptr(v.codes), ptr(v.unit), n, g, hd), _PageTable(ptr(table), table.shape[0], table.shape[1])


@_on_device
def append8(qkv, k: Pages8, v: Pages8, table, q_out, *, heads, dim, vdim, q_norm, k_norm, eps, freqs, n_rot, positions=None, slots=None, portions: Portions8 | None = None,
            head_norm=False, v_off=None, mscale=1.0, maps=1, append=True, pdl=False) -> None:
    """Norm of q and k, rotation, q to padded fp32 rows [rows, H, 64 or 128], k and v into the cache; arguments as of :func:`rows.paged_append`.  Rows are one token a
    sequence at ``positions`` of ``slots`` (of rows of one slot the later ones are appended after the earlier ones), or those of ``portions``."""
    dev, w = qkv.device, "append8"
    c, t = _cache(w, k, v, table, dev)
    n, G = qkv.shape[0], c.kv_heads
    _need(w, "qkv", qkv, torch.float32, dev, None, None, contiguous=False)
    _need(w, "q_out", q_out, torch.float32, dev, n, heads, c.hd)
    kv = G if append else 0
    v_off = (heads + maps * G) * dim if v_off is None else v_off
    if heads < 1 or heads % G or dim < 1 or vdim < 1 or maps not in (1, 2) or heads % maps or maps * dim > c.hd or vdim > c.hd or v_off < 0 or \
            max((heads + maps * kv) * dim, v_off + G * vdim if append else 0) > qkv.shape[1]:
        raise ValueError(f"{w}: {heads} heads of {dim}, {G} of {vdim} from column {v_off} on, {maps} maps, in {qkv.shape[1]} columns and cache rows of {c.hd}")
    if n_rot < 0 or n_rot > dim or n_rot % 2:
        raise ValueError(f"{w}: {n_rot} rotated dimensions of {dim}")
    if n_rot:
        _need(w, "freqs", freqs, torch.float64, dev, None)
        if len(freqs) < n_rot // 2:
            raise ValueError(f"{w}: {len(freqs)} frequencies for {n_rot} dimensions")
    if (q_norm is None) != (k_norm is None) or (q_norm is not None and (maps > 1 or not append)):
        raise ValueError(f"{w}: norms")
    for name, x, h in (("q_norm", q_norm, heads), ("k_norm", k_norm, G)):
        if x is not None:
            _need(w, name, x, torch.float32, dev, None)
            if len(x) < dim * (1 if head_norm else h):
                raise ValueError(f"{w}: {name} of {len(x)}")
    if (portions is None) == (positions is None):
        raise ValueError(f"{w}: either positions and slots or portions")
    if portions is None:
        _need(w, "positions", positions, torch.int32, dev, n)
        _need(w, "slots", slots, torch.int32, dev, n)
        where = (ptr(positions), ptr(slots), None, 0, 1)
    else:
        if portions.rows > n or portions.segs.device != dev:
            raise ValueError(f"{w}: portions of {portions.rows} rows on {portions.segs.device}")
        where = (None, None, ptr(portions.segs), portions.segs.shape[0], portions.per)
    if not n:
        return
    a = Append8Args(ptr(qkv), qkv.stride(0), n, heads, dim, vdim, ptr(q_norm), ptr(k_norm), eps, ptr(freqs) if n_rot else None, n_rot, *where, t, ptr(q_out), c, int(head_norm),
                    v_off, mscale, maps, int(not append))
    _check(lib().b2_append8(C.byref(a), int(pdl), _stream(qkv)), w)


def read8(k: Pages8, v: Pages8, pages, table, k_out, v_out, pdl=False) -> None:
    """Pages as f16 values, [n, KV heads, 64, columns] each.  ``pages`` [n, 4] int32: slot, page of the slot, rows that are wanted (what lies behind them is written as
    zeros, as are pages that are not there), 0."""
    _read8(pages, k, v, table, k_out, v_out, pdl)


@_on_device
def _read8(pages, k, v, table, k_out, v_out, pdl) -> None:
    dev, w = pages.device, "read8"
    c, t = _cache(w, k, v, table, dev)
    _need(w, "pages", pages, torch.int32, dev, None, 4)
    n = pages.shape[0]
    for name, o in (("k_out", k_out), ("v_out", v_out)):
        _need(w, name, o, torch.float16, dev, n, c.kv_heads, PAGE, c.hd)
    if n:
        _check(lib().b2_read8(C.byref(c), C.byref(t), C.c_void_p(ptr(pages)), n, C.c_void_p(ptr(k_out)), C.c_void_p(ptr(v_out)), int(pdl), _stream(pages)), w)


def _attend(w, q, k, v, table, out, where, vdim, scale, softcap, chunk, window, keep, gate, diff, pdl) -> None:
    dev = q.device
    c, t = _cache(w, k, v, table, dev)
    n, heads = q.shape[:2]
    _need(w, "q", q, torch.float32, dev, None, None, c.hd)
    _need(w, "out", out, (torch.float32, torch.bfloat16), dev, n, None, contiguous=False)
    if heads < 1 or heads % c.kv_heads or not 1 <= vdim <= c.hd or (diff.on and heads // c.kv_heads % 2) or out.shape[1] < (heads // 2 if diff.on else heads) * vdim:
        raise ValueError(f"{w}: {heads} heads on {c.kv_heads} of {vdim} columns into rows of {out.shape[1]}")
    if chunk < 0 or window < 0 or keep < 0 or (chunk and window) or softcap < 0:
        raise ValueError(f"{w}: chunk {chunk}, window {window}, keep {keep}, softcap {softcap}")
    splits = 1
    acc, ml = torch.empty(n, heads, splits, c.hd, device=dev), torch.empty(n, heads, splits, 2, device=dev)
    a = Attn8Args(ptr(q), n, heads, vdim, c, t, *where, chunk, window, keep, scale, softcap, splits, ptr(acc), ptr(ml), ptr(out), out.stride(0),
                  int(out.dtype == torch.bfloat16), gate, diff)
    _check(lib().b2_attn8(C.byref(a), int(pdl), _stream(q)), w)


@_on_device
def attn_decode8(qkv, k: Pages8, v: Pages8, positions, slots, table, out, *, heads, dim, vdim, q_norm, k_norm, eps, freqs, n_rot, scale, n_ctx, softcap=0.0, chunk=0, window=0,
                 keep=0, head_norm=False, v_off=None, mscale=1.0, gate=NO_GATE, maps=1, append=True, diff=NO_DIFF, pdl=False) -> None:
    """Decode attention on raw projections, one token a sequence: what :func:`append8` does, then attention of the rows' positions over the cache, difference of maps and
    gate into rows of ``out``.  ``n_ctx``: most keys that a sequence holds."""
    n = qkv.shape[0]
    q = torch.empty(n, heads, k.codes.shape[3], device=qkv.device)
    append8(qkv, k, v, table, q, heads=heads, dim=dim, vdim=vdim, q_norm=q_norm, k_norm=k_norm, eps=eps, freqs=freqs, n_rot=n_rot, positions=positions, slots=slots,
            head_norm=head_norm, v_off=v_off, mscale=mscale, maps=maps, append=append, pdl=pdl)
    if n:
        _attend("attn_decode8", q, k, v, table, out, (ptr(positions), ptr(slots), None, 0), vdim, scale, softcap, chunk, window, keep, gate, diff, pdl)


@_on_device
def attn_prompt8(q, k: Pages8, v: Pages8, portions: Portions8, table, out, *, vdim, scale, softcap=0.0, chunk=0, window=0, keep=0, gate=NO_GATE, diff=NO_DIFF, pdl=False) -> None:
    """Attention of the rows of ``portions``, whose queries ``q`` [rows, H, 64 or 128] and whose keys and values in the cache :func:`append8` has prepared.  ``portions``
    have to be made with this call's masks."""
    if portions.rows > q.shape[0] or portions.segs.device != q.device:
        raise ValueError(f"attn_prompt8: portions of {portions.rows} rows on {portions.segs.device} for {q.shape[0]} on {q.device}")
    _attend("attn_prompt8", q, k, v, table, out, (None, None, ptr(portions.segs), portions.segs.shape[0]), vdim, scale, softcap, chunk, window, keep, gate, diff, pdl)
