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

import numpy as np
import torch

from .cuda import AttnPrefillArgs, _check, lib
from .rows import NO_DIFF, NO_GATE, AttnPagedArgs, DiffHeads, F, HeadGate, I, P, _st

PAGE = 64
MAX_UNITS = 256                  # sequences of one launch of the attention kernel
f32, bf16, i32 = torch.float32, torch.bfloat16, torch.int32

_Pages8 = _st("_Pages8", [("k", P), ("ku", P), ("v", P), ("vu", P), ("n_pages", I), ("kv_heads", I), ("hd", I)])
_PageTable = _st("_PageTable", [("table", P), ("n_slots", I), ("max_pages", I)])
Append8Args = _st("Append8Args", [("qkv", P), ("ldq", I), ("rows", I), ("n_heads", I), ("dim", I), ("vdim", I), ("q_norm", P), ("k_norm", P), ("eps", F), ("freqs", P),
                                  ("n_rot", I), ("positions", P), ("slots", P), ("segs", P), ("n_segs", I), ("per", I), ("t", _PageTable), ("q_out", P), ("c", _Pages8),
                                  ("head_norm", I), ("v_off", I), ("mscale", F), ("maps", I), ("no_append", I)])
Attn8Args = _st("Attn8Args", [("q", P), ("rows", I), ("n_heads", I), ("vdim", I), ("c", _Pages8), ("t", _PageTable), ("positions", P), ("slots", P), ("segs", P), ("n_segs", I),
                              ("chunk", I), ("window", I), ("keep", I), ("scale", F), ("softcap", F), ("row_tile", I), ("turn", I), ("tiles", I), ("ctas", I), ("part_acc", P), ("part_ml", P), ("out", P),
                              ("ldo", I), ("out16", I), ("gate", HeadGate), ("diff", DiffHeads), ("behind", I)])


@dataclass(frozen=True)
class Pages8:
    """Keys or values of a layer: ``codes`` [pages, KV heads, 64, 64 or 128] uint8, ``unit`` [pages, KV heads] fp32."""

    codes: torch.Tensor
    unit: torch.Tensor

    def __post_init__(self):
        c, u = self.codes, self.unit
        if c.dim() != 4 or c.shape[2] != PAGE or c.shape[3] not in (64, 128) or c.dtype != torch.uint8 or not c.is_contiguous() or not c.shape[0] or not c.shape[1]:
            raise ValueError(f"Pages8: codes {tuple(c.shape)} {c.dtype}")
        if u.shape != c.shape[:2] or u.dtype != f32 or not u.is_contiguous() or u.device != c.device:
            raise ValueError(f"Pages8: units {tuple(u.shape)} {u.dtype} on {u.device}")
        # device and sizes, in the order in which calls need them
        object.__setattr__(self, "_sizes", (c.get_device(), c.shape[0], c.shape[1], c.shape[3]))

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


@dataclass(frozen=True)
class Portions8:
    """Portions of prompts in a step, of different slots: what :func:`append8` and :func:`attn_prompt8` have to know of them.  Int32 tensors on the table's device."""

    segs: torch.Tensor               # [n, 4]: first row, rows, slot, position of the first row
    rows: int                        # of all portions
    per: int                         # most pages that a portion's rows go to
    longest: int                     # most rows of one
    masks: tuple[int, int, int]      # window, keep, chunk
    # for attention on values that are read out first: tiles of 128 (of 64) rows, the pages that they may see, and where each portion's pages are among those
    tiles: torch.Tensor              # [tiles, 4]: first row, rows, portion, position
    half_tiles: torch.Tensor
    pages: torch.Tensor              # [pages, 4]: see read8
    table: torch.Tensor              # [n, pages of a slot]


def portions8(parts, table: torch.Tensor, *, window: int = 0, keep: int = 0, chunk: int = 0) -> Portions8:
    """``parts``: (first row, rows, slot, position of the first row) of each portion, rows one after the other; the masks are those of the attention."""
    n_slots, max_pages = table.shape
    if window < 0 or keep < 0 or chunk < 0 or (chunk and window):
        raise ValueError(f"portions8: chunk {chunk}, window {window}, keep {keep}")
    at, slots = 0, set()
    tiles, halves, pages = [], [], []
    where = np.zeros((len(parts), max_pages), np.int32)
    for i, (row, n, slot, pos) in enumerate(parts):
        if n < 1 or row != at or not 0 <= slot < n_slots or pos < 0 or pos + n > max_pages * PAGE:
            raise ValueError(f"portions8: {n} rows from {row} on at position {pos} of slot {slot}, in a table {tuple(table.shape)}")
        if slot in slots:
            raise ValueError(f"portions8: two portions of slot {slot}")
        at += n
        slots.add(slot)
        tiles += [(row + r, min(128, n - r), i, pos + r) for r in range(0, n, 128)]
        halves += [(row + r, min(64, n - r), i, pos + r) for r in range(0, n, 64)]
        last = (pos + n - 1) // PAGE
        first = (pos - pos % chunk if chunk else max(0, pos - window + 1) if window else 0) // 128 * 2          # tiles of 128 keys
        seen = [*range(0, min(first, -(-keep // 128) * 2) if window else 0), *range(first, last + 1)]
        where[i, seen] = np.arange(len(pages), len(pages) + len(seen))
        pages += [(slot, b, min(PAGE, pos + n - b * PAGE), 0) for b in seen]
    if not at:
        raise ValueError("portions8: no rows")
    lists = [np.asarray(x, np.int32) for x in (parts, tiles, halves, pages, where)]
    flat = torch.from_numpy(np.concatenate([x.reshape(-1) for x in lists])).to(table.device)
    segs, tiles, halves, pages, where = (t.view(x.shape) for t, x in zip(flat.split([x.size for x in lists]), lists))
    return Portions8(segs, at, max((p + n - 1) // PAGE - p // PAGE + 1 for _, n, _, p in parts), max(n for _, n, _, _ in parts), (window, keep, chunk), tiles, halves, pages, where)


def _on_device(f):
    """Run ``f`` with its first tensor's device current."""
    @functools.wraps(f)
    def call(x, *a, **kw):
        dev = x.get_device()
        if dev < 0:
            raise ValueError(f"{f.__name__}: tensors on {x.device}")
        if dev == torch.cuda.current_device():
            return f(x, *a, **kw)
        with torch.cuda.device(dev):
            return f(x, *a, **kw)
    return call


@functools.lru_cache(maxsize=None)
def _entry(name: str):
    f = getattr(lib(), name)
    f.restype, f.argtypes = I, {"b2_append8": [P, I, P], "b2_attn8": [P, I, P], "b2_decode8": [P, P, I, P], "b2_read8": [P, P, P, I, P, P, I, I, P], "b2_attn_prefill_paged": [P, P, I, I, I, P], "b2_attn8_status": []}[name]
    return f


def _stream(dev: int) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


@functools.lru_cache(maxsize=64)
def _sms(dev: int) -> int:
    return torch.cuda.get_device_properties(dev).multi_processor_count


def _refuse(what: str, name: str, t: torch.Tensor | None):
    raise ValueError(f"{what}: {name} " + ("is missing" if t is None else f"{tuple(t.shape)} {t.dtype} on {t.device}, strides {t.stride()}"))


def _flat(what: str, name: str, t: torch.Tensor | None, dtype, dev: int, shape) -> int:
    """Address of a tensor that is one piece, of that type, device and shape."""
    if t is None or t.dtype is not dtype or t.get_device() != dev or t.shape != shape or not t.is_contiguous():
        _refuse(what, name, t)
    return t.data_ptr()


def _vector(what: str, name: str, t: torch.Tensor | None, dtype, dev: int, least: int) -> int:
    """Address of a vector of at least so many elements."""
    if t is None or t.dtype is not dtype or t.get_device() != dev or t.dim() != 1 or t.numel() < least or not t.is_contiguous():
        _refuse(what, name, t)
    return t.data_ptr()


def _cache(what: str, k: Pages8, v: Pages8, table: torch.Tensor, dev: int) -> tuple:
    if k._sizes != v._sizes or k._sizes[0] != dev:
        raise ValueError(f"{what}: keys {tuple(k.codes.shape)} on {k.codes.device}, values {tuple(v.codes.shape)} on {v.codes.device}")
    if table.dtype is not i32 or table.get_device() != dev or table.dim() != 2 or not table.is_contiguous():
        _refuse(what, "table", table)
    return _Pages8(k.codes.data_ptr(), k.unit.data_ptr(), v.codes.data_ptr(), v.unit.data_ptr(), *k._sizes[1:]), _PageTable(table.data_ptr(), *table.shape)


def _append_args(w, dev, c, t, qkv, q_out, n, heads, dim, vdim, q_norm, k_norm, eps, freqs, n_rot, head_norm, v_off, mscale, maps, append, where) -> Append8Args:
    G, hd = c.kv_heads, c.hd
    if qkv.dtype is not f32 or qkv.stride(1) != 1 and qkv.shape[1] != 1:
        _refuse(w, "qkv", qkv)
    cols, v_off = qkv.shape[1], (heads + maps * G) * dim if v_off is None else v_off
    if heads < 1 or heads % G or dim < 1 or vdim < 1 or maps not in (1, 2) or heads % maps or maps * dim > hd or vdim > hd or v_off < 0 or \
            heads * dim > cols or (append and max((heads + maps * G) * dim, v_off + G * vdim) > cols):
        raise ValueError(f"{w}: {heads} heads of {dim}, {G} of {vdim} from column {v_off} on, {maps} maps, in {cols} columns and cache rows of {hd}")
    if n_rot < 0 or n_rot > dim or n_rot % 2:
        raise ValueError(f"{w}: {n_rot} rotated dimensions of {dim}")
    if (q_norm is None) != (k_norm is None) or (q_norm is not None and (maps > 1 or not append)):
        raise ValueError(f"{w}: norms")
    qn = kn = None
    if q_norm is not None:
        qn, kn = _vector(w, "q_norm", q_norm, f32, dev, dim if head_norm else heads * dim), _vector(w, "k_norm", k_norm, f32, dev, dim if head_norm else G * dim)
    return Append8Args(qkv.data_ptr(), qkv.stride(0), n, heads, dim, vdim, qn, kn, eps, _vector(w, "freqs", freqs, torch.float64, dev, n_rot // 2) if n_rot else None, n_rot, *where, t,
                       q_out, c, head_norm, v_off, mscale, maps, not append)


def _attn_args(w, dev, c, t, q, n, heads, where, tiles, acc, ml, ctas, out, vdim, scale, softcap, chunk, window, keep, gate, diff) -> Attn8Args:
    if out.dtype is not bf16 and out.dtype is not f32 or out.get_device() != dev or out.dim() != 2 or out.shape[0] != n or out.stride(1) != 1:
        _refuse(w, "out", out)
    if heads < 1 or heads % c.kv_heads or not 1 <= vdim <= c.hd or (diff.on and heads // c.kv_heads % 2) or out.shape[1] < (heads // 2 if diff.on else heads) * vdim:
        raise ValueError(f"{w}: {heads} heads on {c.kv_heads} of {vdim} columns into rows of {out.shape[1]}")
    if chunk < 0 or window < 0 or keep < 0 or (chunk and window) or softcap < 0:
        raise ValueError(f"{w}: chunk {chunk}, window {window}, keep {keep}, softcap {softcap}")
    return Attn8Args(q, n, heads, vdim, c, t, *where, chunk, window, keep, scale, softcap, *tiles, ctas, acc, ml, out.data_ptr(), out.stride(0),
                     out.dtype is bf16, gate, diff, 0)


def _row_tiles(rows: int) -> tuple[int, int, int]:
    """Where a sequence has so many rows for the heads of a KV head: (query rows and keys that are taken together, tiles of the rows)."""
    tile = 8 if rows <= 8 else 16 if rows <= 16 else 128
    return tile, 128 if tile == 128 else 32, -(-rows // tile)


def _pieces(c, tiles, units: int, dev: int) -> tuple[int, int]:
    """(CTAs that fit the GPU at once, rows of partial results: those of as many CTAs, and of one more for each item)."""
    ctas = _sms(dev) * (2 if tiles[0] == 8 else 1)
    return ctas, (min(units, MAX_UNITS) * tiles[2] * c.kv_heads + ctas) * tiles[0]


@_on_device
def append8(qkv, k: Pages8, v: Pages8, table, q_out, *, heads, dim, vdim, q_norm, k_norm, eps, freqs, n_rot, positions=None, slots=None, portions: Portions8 | None = None,
            head_norm=False, v_off=None, mscale=1.0, maps=1, append=True, pdl=False) -> None:
    """Norm of q and k, rotation, q to padded fp32 rows [rows, H, 64 or 128], k and v into the cache; arguments as of :func:`rows.paged_append`.  Rows are one token a
    sequence at ``positions`` of ``slots`` (of rows of one slot the later ones are appended after the earlier ones), or those of ``portions``."""
    w, dev = "append8", qkv.get_device()
    c, t = _cache(w, k, v, table, dev)
    if qkv.dim() != 2:
        _refuse(w, "qkv", qkv)
    n = qkv.shape[0]
    if (portions is None) == (positions is None):
        raise ValueError(f"{w}: either positions and slots or portions")
    if portions is None:
        where = (_flat(w, "positions", positions, i32, dev, (n,)), _flat(w, "slots", slots, i32, dev, (n,)), None, 0, 1)
    else:
        if portions.rows > n or portions.segs.get_device() != dev:
            raise ValueError(f"{w}: portions of {portions.rows} rows on {portions.segs.device}")
        where = (None, None, portions.segs.data_ptr(), portions.segs.shape[0], portions.per)
    a = _append_args(w, dev, c, t, qkv, _flat(w, "q_out", q_out, f32, dev, (n, heads, c.hd)), n, heads, dim, vdim, q_norm, k_norm, eps, freqs, n_rot, head_norm, v_off, mscale, maps,
                     append, where)
    if n:
        _check(_entry("b2_append8")(C.byref(a), pdl, _stream(dev)), w)


def read8(k: Pages8, v: Pages8, pages, table, k_out, v_out, pdl=False) -> None:
    """Pages as f16 values, [n, KV heads, 64, columns] each.  ``pages`` [n, 4] int32: slot, page of the slot, rows that are wanted (what lies behind them is written as
    zeros, as are pages that are not there), 0."""
    _read8(pages, k, v, table, k_out, v_out, pdl)


@_on_device
def _read8(pages, k, v, table, k_out, v_out, pdl) -> None:
    w, dev = "read8", pages.get_device()
    c, t = _cache(w, k, v, table, dev)
    n = pages.shape[0]
    at = _flat(w, "pages", pages, i32, dev, (n, 4))
    shape = (n, c.kv_heads, PAGE, c.hd)
    out = _flat(w, "k_out", k_out, torch.float16, dev, shape), _flat(w, "v_out", v_out, torch.float16, dev, shape)
    if n:
        _check(_entry("b2_read8")(C.byref(c), C.byref(t), at, n, *out, False, pdl, _stream(dev)), w)


@_on_device
def attn_decode8(qkv, k: Pages8, v: Pages8, positions, slots, table, out, *, heads, dim, vdim, q_norm, k_norm, eps, freqs, n_rot, scale, n_ctx, softcap=0.0, chunk=0, window=0,
                 keep=0, head_norm=False, v_off=None, mscale=1.0, gate=NO_GATE, maps=1, append=True, diff=NO_DIFF, pdl=False) -> None:
    """Decode attention on raw projections, one token a sequence: what :func:`append8` does, then attention of the rows' positions over the cache, difference of maps and
    gate into rows of ``out``.  ``n_ctx``: most keys that a sequence holds."""
    w, dev = "attn_decode8", qkv.get_device()
    c, t = _cache(w, k, v, table, dev)
    if qkv.dim() != 2:
        _refuse(w, "qkv", qkv)
    n = qkv.shape[0]
    at, sl = _flat(w, "positions", positions, i32, dev, (n,)), _flat(w, "slots", slots, i32, dev, (n,))
    # rotated queries, partial results, their statistics
    tiles = _row_tiles(heads // c.kv_heads)
    nq, (ctas, pieces) = n * heads * c.hd, _pieces(c, tiles, n, dev)
    ws = torch.empty(nq + pieces * (c.hd + 2), device=qkv.device)
    q = ws.data_ptr()
    p = _append_args(w, dev, c, t, qkv, q, n, heads, dim, vdim, q_norm, k_norm, eps, freqs, n_rot, head_norm, v_off, mscale, maps, append, (at, sl, None, 0, 1))
    a = _attn_args(w, dev, c, t, q, n, heads, (at, sl, None, 0), tiles, q + 4 * nq, q + 4 * (nq + pieces * c.hd), ctas, out, vdim, scale, softcap, chunk, window, keep, gate, diff)
    if n:
        _check(_entry("b2_decode8")(C.byref(p), C.byref(a), pdl, _stream(dev)), w)


@_on_device
def attn_prompt8(q, k: Pages8, v: Pages8, portions: Portions8, table, out, *, vdim, scale, softcap=0.0, chunk=0, window=0, keep=0, gate=NO_GATE, diff=NO_DIFF, pdl=False) -> None:
    """Attention of the rows of ``portions``, whose queries ``q`` [rows, H, 64 or 128] and whose keys and values in the cache :func:`append8` has prepared.  ``portions``
    have to be made with this call's masks."""
    w, dev = "attn_prompt8", q.get_device()
    c, t = _cache(w, k, v, table, dev)
    if q.dim() != 3:
        _refuse(w, "q", q)
    n, heads, _ = q.shape
    at = _flat(w, "q", q, f32, dev, (n, heads, c.hd))
    segs = portions.segs
    if portions.rows > n or segs.get_device() != dev or portions.masks != (window, keep, chunk) or portions.table.shape[1] != table.shape[1]:
        raise ValueError(f"{w}: portions of {portions.rows} rows on {segs.device} with window, keep, chunk {portions.masks} for {n} on {q.device} with {(window, keep, chunk)}")
    units = segs.shape[0]
    tiles = _row_tiles(portions.longest * (heads // c.kv_heads))
    ctas, pieces = _pieces(c, tiles, units, dev)
    a = _attn_args(w, dev, c, t, at, n, heads, (None, None, segs.data_ptr(), units), tiles, 0, 0, ctas, out, vdim, scale, softcap, chunk, window, keep, gate, diff)
    if _reads_out(portions, heads, c.kv_heads) and _attn_read(w, dev, a, portions, q, out, pdl):
        return
    ws = torch.empty(pieces * (c.hd + 2), device=q.device)
    a.part_acc, a.part_ml = ws.data_ptr(), ws.data_ptr() + 4 * pieces * c.hd
    _check(_entry("b2_attn8")(C.byref(a), pdl, _stream(dev)), w)


def _reads_out(portions: Portions8, heads: int, kv_heads: int) -> bool:
    """Whether the pages are read out to f16 first."""
    return portions.longest * (heads // kv_heads) > 256


def _attn_read(w, dev, a: Attn8Args, portions: Portions8, q, out, pdl) -> bool:
    """Attention on tcgen05 over the portions' pages as f16 values; False: not taken, nothing launched."""
    c, diff = a.c, a.diff.on
    if not a.out16 or a.out % 16 or (diff and a.gate.kind):
        return False
    pages, tiles = portions.pages, portions.half_tiles if diff else portions.tiles
    n = pages.shape[0]
    k, v = torch.empty(2, n, c.kv_heads, PAGE, c.hd, device=q.device, dtype=torch.float16)
    _check(_entry("b2_read8")(C.byref(c), C.byref(a.t), pages.data_ptr(), n, k.data_ptr(), v.data_ptr(), True, pdl, _stream(dev)), w)
    p = AttnPrefillArgs(a.q, k.data_ptr(), v.data_ptr(), a.out, None, a.rows, a.n_heads, c.kv_heads, 0, 0, 0, 0, 1, 0, a.scale, a.softcap, None, None)
    pg = AttnPagedArgs(tiles.data_ptr(), portions.table.data_ptr(), portions.table.shape[1], a.chunk, a.vdim, a.ldo, a.window, a.keep, a.gate, a.diff)
    _check(_entry("b2_attn_prefill_paged")(C.byref(p), C.byref(pg), c.hd, tiles.shape[0], n, _stream(dev)), w)
    return True


def status() -> int:
    """0, or 1 once a wait of an attention kernel has run out since the last call; synchronises."""
    return _entry("b2_attn8_status")()
