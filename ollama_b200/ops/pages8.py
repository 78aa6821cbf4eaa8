"""The 8-bit paged cache of attention layers: rows appended to it, its pages read back, attention over it (kernels/pages8.cu, attn_pages8.cu).

Keys and values stand in pages of 64 positions, [page, KV head, position, column], as E4M3 numbers (:class:`Pages8`).  Each page has a unit for each KV head, a power
of two between 2^-15 and 2^7; a value is its number times the unit, and always an f16 number too.  The unit is the least with which the largest magnitude that was
appended to the page fits; larger magnitudes than 57344 become that.  Where an appended row makes the unit grow, the page's other rows are rounded to the new one, and a
row at a page's first position begins the page anew.  Rows have 64 or 128 columns; heads of fewer leave zeros behind theirs.

Tables of pages are [slots, pages] int32: entry i of a slot is the page of its positions 64 i .. 64 i + 63.  Rows whose position is negative hold no token: nothing is
appended for them and their results are left as they are.  So are rows whose slot or position the table does not have.  Where a table's entry is no page of the cache
nothing is appended and nothing outside the cache is read; what attention makes of such positions is not defined.  A page that rows are appended to may be in one slot's
table only, others may be in several.  All calls run on the current stream of the tensors' device.
"""
from __future__ import annotations

import ctypes as C
import importlib.util
import threading
from dataclasses import dataclass

import numpy as np
import torch

from .cuda import AttnPrefillArgs, CudaKernelError, _check, lib
from .rows import NO_DIFF, NO_GATE, AttnPagedArgs, I, P

PAGE = 64
TOGETHER = 1024                  # pages: see portions8
LIFT = 7.0                       # weights of attention on read-out pages count from 2^7 on, as those of the other forms (attn_pages8.cu)


@dataclass(frozen=True)
class Pages8:
    """Keys or values of a layer: ``codes`` [pages, KV heads, 64, 64 or 128] uint8, ``unit`` [pages, KV heads] fp32."""

    codes: torch.Tensor
    unit: torch.Tensor

    def __post_init__(self):
        c, u = self.codes, self.unit
        if c.dim() != 4 or c.shape[2] != PAGE or c.shape[3] not in (64, 128) or c.dtype != torch.uint8 or not c.is_contiguous() or not c.shape[0] or not c.shape[1]:
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


@dataclass(frozen=True)
class Portions8:
    """Portions of prompts in a step, of different slots: what :func:`append8` and :func:`attn_prompt8` have to know of them.  Int32 tensors on the table's device."""

    segs: torch.Tensor               # [n, 4]: first row, rows, slot, position of the first row
    rows: int                        # of all portions
    per: int                         # most pages that a portion's rows go to
    longest: int                     # most rows of one
    masks: tuple[int, int, int]      # window, keep, chunk
    sizes: tuple                     # (rows, keys that they may see, group) of each
    # for attention on values that are read out first: tiles of 128 (of 64) rows, the pages that they may see, and where each portion's pages are among those of its group;
    # a group is what is read out together: from which tile, half tile and page to which
    groups: tuple
    tiles: torch.Tensor              # [tiles, 4]: first row, rows, portion, position
    half_tiles: torch.Tensor
    pages: torch.Tensor              # [pages, 4]: see read8
    table: torch.Tensor              # [n, pages of a slot]

    @property
    def nbytes(self) -> int:
        return sum(t.nbytes for t in (self.segs, self.tiles, self.half_tiles, self.pages, self.table))


def portions8(parts, table: torch.Tensor, *, window: int = 0, keep: int = 0, chunk: int = 0, together: int = TOGETHER) -> Portions8:
    """``parts``: (first row, rows, slot, position of the first row) of each portion, rows one after the other; the masks are those of the attention.  ``together``: most pages
    that attention which reads pages out first holds as f16 values at a time (4 * 64 bytes each for every KV head and column), or those of one slot where they are more; what takes
    more goes in passes."""
    n_slots, max_pages = table.shape
    if window < 0 or keep < 0 or chunk < 0 or (chunk and window):
        raise ValueError(f"portions8: chunk {chunk}, window {window}, keep {keep}")
    at, slots, most = 0, set(), max(together, max_pages)
    tiles, halves, pages, sizes, ends, begins = [], [], [], [], [], (0, 0, 0)
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
        if len(pages) + len(seen) - begins[2] > most:      # a group ends before this portion, whose tiles are in the lists already
            ends.append(begins := (len(tiles) - -(-n // 128), len(halves) - -(-n // 64), len(pages)))
        sizes.append((n, len(seen) * PAGE, len(ends)))
        where[i, seen] = np.arange(len(pages) - begins[2], len(pages) - begins[2] + len(seen))
        pages += [(slot, b, min(PAGE, pos + n - b * PAGE), 0) for b in seen]
    if not at:
        raise ValueError("portions8: no rows")
    ends.append((len(tiles), len(halves), len(pages)))
    groups = tuple(zip(((0, 0, 0), *ends), ends))
    lists = [np.asarray(x, np.int32) for x in (parts, tiles, halves, pages, where)]
    flat = torch.from_numpy(np.concatenate([x.reshape(-1) for x in lists])).to(table.device)
    segs, tiles, halves, pages, where = (t.view(x.shape) for t, x in zip(flat.split([x.size for x in lists]), lists))
    return Portions8(segs, at, max((p + n - 1) // PAGE - p // PAGE + 1 for _, n, _, p in parts), max(n for n, _, _ in sizes), (window, keep, chunk), tuple(sizes), groups,
                     tiles, halves, pages, where)


def _module():
    """The module of the calls (pages8_call.cpp), built where there is none of these sources."""
    from ..kernels.build import build_calls
    spec = importlib.util.spec_from_file_location("ollama_b200.ops._pages8", build_calls())
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _bind(m) -> None:
    """Hands it the kernel library's entry points."""
    try:
        layout = lib().b2_pages8_layout
    except AttributeError:
        raise RuntimeError("the kernel library is older than the calls: run python -m ollama_b200.kernels.build") from None
    layout.restype = C.c_ulonglong
    m.bind(*(C.cast(getattr(lib(), n), C.c_void_p).value for n in ("b2_append8", "b2_attn8", "b2_decode8", "b2_read8")), CudaKernelError, layout())


def _calls():
    m = _module()
    _bind(m)
    return m


_LOADING = threading.Lock()


def load() -> None:
    """Makes the calls ready, building what is missing: before a model's first step rather than in it.  Of several threads one does."""
    with _LOADING:
        if "append8" not in globals():
            m = _calls()
            globals().update(append8=m.append8, read8=m.read8, attn_decode8=m.attn_decode8, _attn_prompt8=m.attn_prompt8)


def __getattr__(name: str):
    """The calls, when one is first asked for."""
    if name not in ("append8", "read8", "attn_decode8", "_attn_prompt8"):
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    load()
    return globals()[name]


def attn_prompt8(q, k: Pages8, v: Pages8, portions: Portions8, table, out, *, vdim, scale, softcap=0.0, chunk=0, window=0, keep=0, gate=NO_GATE, diff=NO_DIFF, pdl=False) -> int:
    """Attention of the rows of ``portions``, whose queries ``q`` [rows, H, 64 or 128] and whose keys and values in the cache :func:`append8` has prepared.  ``portions``
    have to be made with this call's masks.  Returns the launches.

    Queries and weights are rounded to f16 (2^-11 each) whatever type ``out`` has, so queries beyond 65504 have no result; the scores' and weights' sums are 32-bit ones.  Soft
    caps and gates use the fast exponential and quotient, some 2^-21.  Results of many rows, which may be of read-out pages, are within the same bounds."""
    here = globals()
    call = here.get("_attn_prompt8") or __getattr__("_attn_prompt8")
    mask = dict(vdim=vdim, scale=scale, softcap=softcap, chunk=chunk, window=window, keep=keep, gate=gate, diff=diff, pdl=pdl)
    if n := call(q, k, v, portions, table, out, **mask):
        return n
    # many rows: the pages that they may see as f16 values, for attention on tcgen05
    n, heads, hd = q.shape
    kv_heads, tiles, of = k.codes.shape[1], portions.half_tiles if diff.on else portions.tiles, 1 if diff.on else 0
    try:
        wide = torch.empty(2, max(b[2] - a[2] for a, b in portions.groups), kv_heads, PAGE, hd, device=q.device, dtype=torch.float16)
    except torch.OutOfMemoryError:          # the other forms take more time and little memory
        return call(q, k, v, portions, table, out, read_out=False, **mask)
    f = lib().b2_attn_prefill_paged
    f.argtypes = [P, P, I, I, I, I, P]
    a = AttnPrefillArgs(q.data_ptr(), wide[0].data_ptr(), wide[1].data_ptr(), out.data_ptr(), None, n, heads, kv_heads, 0, 0, 0, 0, 1, 0, scale, softcap, None, None)
    for begin, end in portions.groups:
        pages, some = portions.pages[begin[2]:end[2]], tiles[begin[of]:end[of]]
        m = pages.shape[0]
        here["read8"](k, v, pages, table, wide[0, :m], wide[1, :m], pdl, clean=True)
        pg = AttnPagedArgs(some.data_ptr(), portions.table.data_ptr(), portions.table.shape[1], chunk, vdim, out.stride(0), window, min(keep, portions.table.shape[1] * PAGE), gate, diff, LIFT)
        with torch.cuda.device(q.device):
            _check(f(C.addressof(a), C.addressof(pg), hd, some.shape[0], m, 1, torch.cuda.current_stream().cuda_stream), "attn_prompt8")
    return 2 * len(portions.groups)


def status() -> int:
    """0, or 1 once a wait of an attention kernel has run out since the last call; synchronises."""
    return lib().b2_attn8_status()
