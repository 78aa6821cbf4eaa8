"""The 8-bit paged cache in 64 bits: what rows become in it, and attention over what it holds."""
import math

import torch

PAGE, LOW, HIGH, TOP = 64, -15, 7, 448.0
F64 = torch.float64


def e4m3(x):
    """Nearest E4M3 numbers, ties to even."""
    a = x.abs().clamp(max=TOP)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.sign(x) * torch.round(a / step) * step


def unit_for(top):
    """Least power of two within the limits in whose units magnitude ``top`` is at most 448."""
    u = torch.full_like(top, 2.0 ** HIGH)
    for e in range(HIGH - 1, LOW - 1, -1):
        u = torch.where(top <= TOP * 2.0 ** e, 2.0 ** e, u)
    return u


def normed(x, w, eps, head_norm):
    """x [rows, heads, dim]; w [heads * dim] or, for each head, [dim]."""
    if w is None:
        return x
    over = (-1,) if head_norm else (-2, -1)
    y = x / (x.square().mean(over, keepdim=True) + eps).sqrt()
    return y * (w.double() if head_norm else w.double().view(x.shape[1:]))


def rotated(x, pos, freqs, magnitude=1.0):
    """Half-split rotation of the first 2 len(freqs) dimensions."""
    n = len(freqs)
    a = pos.double()[:, None, None] * freqs.double()
    c, s = torch.cos(a) * magnitude, torch.sin(a) * magnitude
    lo, hi = x[..., :n], x[..., n:2 * n]
    return torch.cat([lo * c - hi * s, hi * c + lo * s, x[..., 2 * n:]], -1)


class Cache:
    """Codes (as numbers) and units of keys or values, [pages, heads, 64, columns] and [pages, heads]."""

    def __init__(self, numbers, unit):
        self.n, self.u = numbers.double().clone(), unit.double().clone()

    def values(self):
        return self.n * self.u[..., None, None]

    def append(self, table, slot, pos, x):
        """Rows x [n, heads, columns] at positions pos .. pos + n - 1 of a slot."""
        x = torch.nn.functional.pad(x, (0, self.n.shape[3] - x.shape[2]))
        for b in range(pos // PAGE, (pos + len(x) - 1) // PAGE + 1):
            lo, hi = max(pos, b * PAGE), min(pos + len(x), (b + 1) * PAGE)
            y, p = x[lo - pos:hi - pos].transpose(0, 1), int(table[slot, b])
            new = unit_for(torch.nan_to_num(y.abs(), nan=0.0, posinf=1e30).amax((1, 2)))
            if lo % PAGE:
                new = torch.maximum(new, self.u[p])
                grown = (new > self.u[p])[:, None, None]
                self.n[p] = torch.where(grown, e4m3(self.n[p] * (self.u[p] / new)[:, None, None]), self.n[p])
            self.u[p] = new
            self.n[p, :, lo % PAGE:lo % PAGE + hi - lo] = e4m3((y / new[:, None, None]).clamp(-TOP, TOP))


def visible(pos, n_keys, chunk=0, window=0, keep=0):
    """[rows, keys]: which keys the queries at ``pos`` see."""
    at, p = torch.arange(n_keys), pos.cpu().long()[:, None]
    low = p - p % chunk if chunk else (p - window + 1).clamp(min=0) if window else torch.zeros_like(p)
    return (at <= p) & ((at >= low) | (at < (keep if window else 0)))


def attend(q, k, v, seen, scale, softcap=0.0):
    """q [rows, heads, dim], k, v [kv heads, keys, columns], in 64 bits -> (results, bound of what rounding q to f16 moves a score by)."""
    H, G = q.shape[1], k.shape[0]
    v = torch.where(seen.any(0).to(v.device)[None, :, None], v, 0.0)
    k = torch.where(seen.any(0).to(v.device)[None, :, None], k, 0.0)
    k, v = k.repeat_interleave(H // G, 0), v.repeat_interleave(H // G, 0)
    s = torch.einsum("rhd,hkd->hrk", q, k) * scale
    moved = torch.einsum("rhd,hkd->hrk", q.abs(), k.abs()) * abs(scale) * 2.0 ** -11
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    seen = seen.to(s.device)
    p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
    return torch.einsum("hrk,hkd->rhd", p, v), moved.masked_fill(~seen, 0.0).amax(-1).t()[..., None]


def tolerance(o, moved, v_max, out_dtype):
    """Bound of |got - o|: scores off by ``moved`` move weights by twice that, weights are rounded to f16 (2^-11), sums are 32-bit (counted with the weights, doubled), the
    result to its type (half a step)."""
    last = 2.0 ** -8 if out_dtype == torch.bfloat16 else 2.0 ** -24
    return (2 * moved + 2 * 2.0 ** -11) * v_max * (1 + last) + o.abs() * last + 1e-6 * v_max
