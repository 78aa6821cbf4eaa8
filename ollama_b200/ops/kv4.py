"""The 4-bit K/V cache: rows appended to it and read back, single tokens' and prompts' attention over it, and attention of packed prompts over 16-bit keys and values (kernels/kv4.cu, attn_kv4.cu,
attn_packed.cu).

A layer's keys or values are a :class:`Cache4`: for every 32 columns of a row an f16 scale d and 32 integers 0 .. 15, whose values are d (integer - 8).  d is minus an eighth of the value of largest
magnitude (of two, the negative one), so that one is held to f16's precision and the others within half a step of |d|, one of the other sign that is as large within a step.  Magnitudes beyond
65504 become that, values that are no number zero.  Four and a half bits a value: 0.28 of f16.  Heads have 64 or 128 columns.

All calls run on the current stream of the tensors' device.  Their workspaces come from torch's allocator, so calls on several streams, and captured ones, have their own.
"""
from __future__ import annotations

import ctypes as C
import importlib.util
import threading
from dataclasses import dataclass

import torch

from .cuda import CudaKernelError, lib

BLOCK = 32
TILE = 128                       # keys, and query rows times heads, that attention of prompts takes at a time
TOP = 8188.0                     # largest scale


@dataclass(frozen=True)
class Cache4:
    """Keys or values of a layer: ``codes`` [slots, KV heads, positions, columns / 2] uint8, two integers a byte in the order that kernels/kv4.cuh says, ``scale`` [slots, KV heads, positions,
    columns / 32] f16."""

    codes: torch.Tensor
    scale: torch.Tensor

    def __post_init__(self):
        c, s = self.codes, self.scale
        if c.dim() != 4 or c.shape[3] not in (32, 64) or c.dtype != torch.uint8 or not c.is_contiguous() or not c.numel():
            raise ValueError(f"Cache4: codes {tuple(c.shape)} {c.dtype}")
        if s.shape != (*c.shape[:3], c.shape[3] // 16) or s.dtype != torch.float16 or not s.is_contiguous() or s.device != c.device:
            raise ValueError(f"Cache4: scales {tuple(s.shape)} {s.dtype} on {s.device}")

    @classmethod
    def empty(cls, slots: int, kv_heads: int, n_ctx: int, dim: int, device="cuda") -> "Cache4":
        """Rows of zeros."""
        if dim not in (64, 128):
            raise ValueError(f"Cache4: heads of {dim} columns")
        return cls(torch.full((slots, kv_heads, n_ctx, dim // 2), 0x88, device=device, dtype=torch.uint8), torch.zeros(slots, kv_heads, n_ctx, dim // BLOCK, device=device, dtype=torch.float16))

    @property
    def shape(self) -> tuple[int, int, int, int]:
        """(slots, KV heads, positions, columns)."""
        return (*self.codes.shape[:3], 2 * self.codes.shape[3])


def encode4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of rows [..., 64 or 128] in tensor operations, on any device: what :func:`append4` makes of them, but for quotients within 2^-23 of a border between two codes, which it takes by the
    reciprocal."""
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=torch.inf, neginf=-torch.inf).unflatten(-1, (-1, BLOCK))
    hi, lo = x.amax(-1), x.amin(-1)
    d = (torch.where(hi > -lo, hi, lo) * -0.125).clamp(-TOP, TOP).to(torch.float16)
    w = d.float()[..., None]
    c = torch.where(w != 0, torch.round(x / w) + 8, 8.0).clamp(0, 15).to(torch.uint8)
    c = c.unflatten(-1, (4, 4, 2)).transpose(-4, -3).transpose(-1, -2)              # [..., word, block, odd, pair]
    return (c[..., 0::2] | c[..., 1::2] << 4).flatten(-4).contiguous(), d


def decode4(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """Rows [..., 64 or 128] in fp32, in tensor operations."""
    c = codes.unflatten(-1, (4, -1, 2, 2))                                          # [..., word, block, odd, byte]
    c = torch.stack([c & 15, c >> 4], -1).flatten(-2).transpose(-1, -2).transpose(-4, -3).flatten(-3)
    return ((c.float() - 8) * scale.float()[..., None]).flatten(-2)


@dataclass(frozen=True)
class Portions4:
    """Rows of several sequences in a step, for :func:`attn_prompt4` and :func:`attn_packed`: what a model makes once for a step of all its layers."""

    tiles: torch.Tensor              # [n, 12] int32: first row, rows, slot, position, cache row of position 0, key tiles from .. to, partial result or -1, KV head
    merges: torch.Tensor             # [m, 8] int32: first row, rows, first partial result, partial results, KV head
    starts: torch.Tensor             # [CTAs + 1] int32: CTA i takes tile i, then starts[i] .. starts[i + 1] - 1
    rows: int                        # of all portions
    parts: int                       # partial results
    merge_rows: int                  # rows of theirs that the largest sum has
    window: int
    group: int                       # query heads a KV head
    cache: tuple[int, int, int, int]


def portions4(parts, heads: int, k, *, window: int = 0) -> Portions4:
    """``parts``: (first row, rows, slot, position of the first row) of each portion, rows one after the other, and where that is not 0 the cache row of the sequence's position 0 behind it.
    ``heads`` query heads attend over ``k``, a :class:`Cache4` or 16-bit keys [slots, KV heads, positions, columns], with the attention's ``window``.  Where keys are cut follows from all
    portions, so a row's result beside other portions is that of the row alone but for roundings."""
    slots, kv_heads, n_ctx, dim = k.shape
    if heads < 1 or heads % kv_heads or heads // kv_heads > TILE or window < 0:
        raise ValueError(f"portions4: {heads} heads on {kv_heads}, window {window}")
    at, rows = 0, []
    for row, n, slot, pos, *more in parts:
        base = more[0] if more else 0
        if n < 1 or row != at or not 0 <= slot < slots or pos < 0 or base < 0 or base + pos + n > n_ctx:
            raise ValueError(f"portions4: {n} rows from {row} on at position {pos} of slot {slot}, from row {base} on, in a cache of {slots} slots of {n_ctx}")
        at += n
        rows.append((row, n, slot, pos, base))
    if not at:
        raise ValueError("portions4: no rows")
    dev = k.codes.device if isinstance(k, Cache4) else k.device
    sms = torch.cuda.get_device_properties(dev).multi_processor_count if dev.type == "cuda" else 148
    here = globals()
    *lists, n_parts, merge_rows = (here.get("_plan") or __getattr__("_plan"))(torch.tensor(rows, dtype=torch.int32), heads // kv_heads, kv_heads, window, sms)
    flat = torch.cat([x.view(-1) for x in lists]).to(dev)
    tiles, merges, starts = (t.view(x.shape) for t, x in zip(flat.split([x.numel() for x in lists]), lists))
    return Portions4(tiles, merges, starts.view(-1), at, n_parts, merge_rows, window, heads // kv_heads, (slots, kv_heads, n_ctx, dim))


CALLS = ("append4", "read4", "attn_decode4", "attn_step4", "attn_prompt4", "attn_packed")
_LOADING = threading.Lock()


def _module():
    """The module of the calls (kv4_call.cpp), built where there is none of these sources."""
    from ..kernels.build import build_calls
    spec = importlib.util.spec_from_file_location("ollama_b200.ops._kv4", build_calls(what="kv4"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _bind(m) -> None:
    """Hands it the kernel library's entry points."""
    try:
        layout = lib().b2_kv4_layout
    except AttributeError:
        raise RuntimeError("the kernel library is older than the calls: run python -m ollama_b200.kernels.build") from None
    layout.restype = C.c_ulonglong
    m.bind(*(C.cast(getattr(lib(), n), C.c_void_p).value for n in ("b2_append4", "b2_read4", "b2_attn4", "b2_attn4_room", "b2_attn_packed")), CudaKernelError, layout())


def load() -> None:
    """Makes the calls ready, building what is missing: before a model's first step rather than in it.  Of several threads one does."""
    with _LOADING:
        if CALLS[0] not in globals():
            m = _module()
            _bind(m)
            globals().update({n: getattr(m, n) for n in CALLS}, _plan=m.plan)


def __getattr__(name: str):
    """The calls, when one is first asked for."""
    if name not in (*CALLS, "_plan"):
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    load()
    return globals()[name]


def status() -> int:
    """0, or 1 once a wait of the prompts' kernel has run out since the last call; synchronises."""
    return lib().b2_attn_packed_status()
