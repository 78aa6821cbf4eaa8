"""The 4-bit cache in 64 bits: what rows become in it, what its bytes say, and attention over it."""
import math

import torch

F64 = torch.float64
HALF16, HALFB = 2.0 ** -11, 2.0 ** -8           # largest relative roundings to f16, to bf16
TOP = 8188.0


def held(codes, scale):
    """Values [..., columns] of rows, column by column from their bits."""
    d = 2 * codes.shape[-1]
    out = torch.empty(*codes.shape[:-1], d, dtype=F64, device=codes.device)
    for col in range(d):
        block, word, pair, odd = col // 32, col % 32 // 8, col % 8 // 2, col % 2
        byte = codes[..., 4 * (word * (d // 32) + block) + 2 * odd + pair // 2].long()
        out[..., col] = ((byte >> 4 * (pair % 2) & 15) - 8) * scale[..., block].double()
    return out


def scales(x):
    """Exact scales of rows [..., columns] before they are rounded to f16."""
    x = torch.nan_to_num(x, nan=0.0, posinf=1e30, neginf=-1e30).unflatten(-1, (-1, 32))
    hi, lo = x.amax(-1), x.amin(-1)
    return (-torch.where(hi > -lo, hi, lo) / 8).clamp(-TOP, TOP)


def rounded(x):
    """Rows [..., columns] as the cache holds them."""
    d = scales(x.double()).to(torch.float16).double()[..., None]
    y = torch.nan_to_num(x.double(), nan=0.0, posinf=1e30, neginf=-1e30).unflatten(-1, (-1, 32))
    return torch.where(d == 0, 0.0, d * torch.round(y / torch.where(d == 0, 1.0, d)).clamp(-8, 7)).flatten(-2)


def assert_held(x, codes, scale, off=0.0):
    """Rows that hold ``x`` [..., columns] (64 bits; the kernel's own may be ``off`` of the row's largest value away): f16-rounded scales, and codes that are the nearest but for those so near a border."""
    x, codes, scale = x.cpu(), codes.cpu(), scale.cpu()
    d, want = scale.double(), scales(x)
    big = want.abs().amax(-1, keepdim=True)
    # opposite extremes that are closer than `off` may go either way
    y = x.unflatten(-1, (-1, 32))
    tie = (y.amax(-1) + y.amin(-1)).abs() <= 16 * off * big
    err = torch.where(tie, (d.abs() - want.abs()).abs(), (d - want).abs())
    assert (err <= HALF16 * want.abs() + off * big + 2.0 ** -25).all(), float(err.max())
    got = held(codes, scale).unflatten(-1, (-1, 32))
    q = torch.where(d[..., None] == 0, 0.0, y / torch.where(d == 0, 1.0, d)[..., None])
    near = (got - y).abs() <= d.abs()[..., None] * (0.5 + 1e-5) + 8 * off * big[..., None] + torch.where(d == 0, 2.0 ** -22, 0.0)[..., None]
    last = (got == 7 * d[..., None]) & (q >= 7.5 - 1e-3) | (got == -8 * d[..., None]) & (q <= -8.5 + 1e-3)
    assert (near | last).all()


def normed(x, w, eps):
    return x if w is None else x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double().cpu()


def rotated(x, pos, inv_freq, n_rot, neox, mscale=1.0):
    """x [rows, heads, columns]."""
    h = n_rot // 2
    a = pos.double().cpu()[:, None, None] * inv_freq.double().cpu()[:h]
    c, s = torch.cos(a) * mscale, torch.sin(a) * mscale
    first = torch.arange(h) * (1 if neox else 2)
    second = first + (h if neox else 1)
    y = x.clone()
    y[..., first], y[..., second] = x[..., first] * c - x[..., second] * s, x[..., second] * c + x[..., first] * s
    return y


def attend(q, keys, vals, pos, *, scale, window=0, softcap=0.0, sinks=None, wide=0.0):
    """Rows q [n, H, D] at positions ``pos`` over keys and values [G, K, D]: results [n, H * D] and how far a kernel's may be from them before their last rounding.

    Queries are rounded to f16 (each score moves by at most 2^-11 of the sum of its products' sizes), weights are (2^-11 of each), ``wide`` is the largest relative rounding of keys and values
    where they are made f16 numbers; a factor e^x on each weight and on their sum moves the mean by at most 2 (e^x - 1) of the mean size; soft caps use a fast tanh, 2^-20 of the cap.  Weights so small that they are f16
    subnormals are rounded by up to 2^-25 where the heaviest (in the 4-bit decode kernel: the heaviest weight times its values' scale) counts 2^6 or more, which moves the mean by at most 2^-31 of the
    largest value for each key."""
    H, G = q.shape[1], keys.shape[0]
    q, keys, vals, dev = q.double(), keys.double(), vals.double(), q.device
    out, err = torch.empty(len(q), H, q.shape[2], dtype=F64, device=dev), torch.empty(len(q), H, q.shape[2], dtype=F64, device=dev)
    at, pos = torch.arange(keys.shape[1], device=dev), pos.to(dev)[:, None]
    seen = (at <= pos) & (at > pos - window) if window else at <= pos
    for h in range(H):
        k, v = keys[h * G // H], vals[h * G // H]
        x = q[:, h] @ k.T * scale
        move = (abs(scale) * (HALF16 + wide) * (q[:, h].abs() @ k.abs().T)).masked_fill(~seen, 0).amax(1)
        if softcap:
            x, move = softcap * torch.tanh(x / softcap), move + softcap * 2.0 ** -20
        x = x.masked_fill(~seen, -math.inf)
        if sinks is not None:
            x = torch.cat([x, sinks[h].double().to(dev).expand(len(q), 1)], 1)
        p = torch.softmax(x, 1)[:, :keys.shape[1]]
        out[:, h] = p @ v
        err[:, h] = (2 * (torch.expm1(move) + HALF16) + wide + 2.0 ** -18)[:, None] * (p @ v.abs()) + (seen.sum(1) * 2.0 ** -31)[:, None] * v.abs().max()
    return out.flatten(1), err.flatten(1)


def assert_near(got, want, err):
    last = {torch.bfloat16: HALFB, torch.float16: HALF16, torch.float32: 2.0 ** -22}[got.dtype]
    off = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all()
    bound = err * (1 + last) + last * want.abs() + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    assert (off <= bound).all(), (float((off / bound).max()), float(off.max()))
