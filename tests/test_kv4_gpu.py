"""The 4-bit cache's kernels and packed prompts against 64 bits (kv4_oracle.py says what the bounds are made of)."""
import threading

import pytest
import torch

import kv4_oracle as O
from ollama_b200.ops import kv4

pytestmark = pytest.mark.gpu
F16, F32, B16 = torch.float16, torch.float32, torch.bfloat16


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def filled(slots, kv_heads, n_ctx, dim, seed=0, spread=2.0):
    """Keys and values of random rows of different sizes, a few columns of which stand out."""
    g, out = gen(seed), []
    for _ in range(2):
        x = torch.randn(slots, kv_heads, n_ctx, dim, device="cuda", generator=g) * torch.exp2((torch.rand(slots, kv_heads, n_ctx, 1, device="cuda", generator=g) - 0.5) * spread)
        x *= 1 + 3 * (torch.rand(dim, device="cuda", generator=g) > 0.94)
        out.append(kv4.Cache4(*kv4.encode4(x)))
    return out


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def values(c, slot=slice(None), upto=None):
    return O.held(c.codes[slot, :, :upto], c.scale[slot, :, :upto])


def freqs(n_rot):
    return (10000.0 ** (-torch.arange(n_rot // 2, dtype=torch.float64) * 2 / max(n_rot, 1))).float().cuda()


# ---- append, read -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv_heads,dim,n_rot,neox,norm,rows", [
    (4, 2, 64, 64, True, False, 1), (4, 2, 64, 64, False, True, 5), (32, 8, 128, 128, True, True, 70), (32, 8, 128, 128, False, False, 16), (7, 1, 128, 64, True, True, 3), (16, 16, 64, 20, True, False, 65),
    (3, 3, 128, 6, True, False, 2), (5, 5, 128, 10, False, True, 66), (1, 1, 64, 0, True, True, 4), (40, 2, 128, 128, True, False, 9), (2, 1, 64, 2, True, False, 1), (12, 12, 128, 12, True, True, 3)])
def test_append_and_read(heads, kv_heads, dim, n_rot, neox, norm, rows):
    g, n_ctx, slots = gen(heads * 131 + rows), 500000, 3
    cols = (heads + 2 * kv_heads) * dim
    n_ctx = 100003 if kv_heads < 8 else 5003
    k, v = (kv4.Cache4.empty(slots, kv_heads, n_ctx, dim) for _ in range(2))
    pos = torch.randperm(n_ctx, device="cuda", generator=g)[:rows].int()
    pos[0] = n_ctx - 1
    slot = torch.randint(0, slots, (rows,), device="cuda", generator=g).int()
    w = [1 + 0.3 * torch.randn(dim, device="cuda", generator=g) for _ in range(2)] if norm else (None, None)
    inv = freqs(n_rot)
    for pitch, lead, kind in ((cols, 0, F32), (cols + 4, 4, F16), (cols + 3, 1, F32)):
        buf = torch.randn(rows, pitch + lead, device="cuda", generator=g)
        qkv = buf[:, lead:lead + cols]
        q_out = torch.full((rows, heads, dim), 7.0, device="cuda", dtype=kind)
        kv4.append4(qkv, k, v, pos, slot, q_out, heads=heads, inv_freq=inv, n_rot=n_rot, neox=neox, mscale=1.3, q_norm=w[0], k_norm=w[1], eps=1e-5)
        x = qkv.double().cpu().view(rows, heads + 2 * kv_heads, dim)
        q, key, val = x.split([heads, kv_heads, kv_heads], 1)
        turn = lambda y, n: O.rotated(O.normed(y, n, 1e-5), pos, inv, n_rot, neox, 1.3)
        # norm, angle, sine and products: some ten roundings of 2^-24 of a row's largest value
        want, off = turn(q, w[0]), 16 * 2.0 ** -24
        size = want.abs().amax(-1, keepdim=True)
        err = (q_out.double().cpu() - want).abs()
        assert (err <= 2 * off * size + (O.HALF16 * want.abs() + 2.0 ** -25 if kind == F16 else 0)).all(), float((err / size).max())
        at = (slot.long(), slice(None), pos.long())
        O.assert_held(turn(key, w[1]), k.codes[at], k.scale[at], 2 * off)
        O.assert_held(val, v.codes[at], v.scale[at], 0.0)
        out = [torch.full((rows, kv_heads, dim), 9.0, device="cuda", dtype=F16) for _ in range(2)]
        kv4.read4(k, v, pos, slot, *out)
        for c, o in zip((k, v), out):
            assert torch.equal(o, O.held(c.codes[at], c.scale[at]).to(F16))
    # without queries the same rows
    before = [t.clone() for c in (k, v) for t in (c.codes, c.scale)]
    kv4.append4(qkv, k, v, pos, slot, heads=heads, inv_freq=inv, n_rot=n_rot, neox=neox, mscale=1.3, q_norm=w[0], k_norm=w[1], eps=1e-5)
    assert all(torch.equal(a, b) for a, b in zip(before, [t for c in (k, v) for t in (c.codes, c.scale)]))


def test_append_of_special_values():
    """Zeros, infinities, no numbers, beyond f16, subnormal scales, opposite extremes: what the tensor form makes of them."""
    x = torch.zeros(8, 3, 128, device="cuda")
    x[1, :, 3], x[1, :, 40], x[2, :, :5], x[2, :, 5] = float("inf"), -float("inf"), float("nan"), 2.0
    x[3], x[3, :, 9], x[4, :, 0], x[4, :, 1], x[5], x[6], x[6, :, 64] = 1e-9, 70000.0, 3.0, -3.0, 2.0 ** -24, 2.0 ** -19, -2.0 ** -17
    x[7] = float("nan")
    k, v = (kv4.Cache4.empty(1, 1, 8, 128) for _ in range(2))
    pos, slot = torch.arange(8, device="cuda", dtype=torch.int32), torch.zeros(8, device="cuda", dtype=torch.int32)
    q = torch.empty(8, 1, 128, device="cuda")
    kv4.append4(x.view(8, 384), k, v, pos, slot, q, heads=1, inv_freq=None, n_rot=0)
    codes, scale = kv4.encode4(x[:, 1:2])
    for c in (k, v):
        assert torch.equal(c.scale[0].transpose(0, 1), scale) and torch.equal(c.codes[0].transpose(0, 1), codes)
    assert torch.equal(q.nan_to_num(nan=5.0), x[:, :1].nan_to_num(nan=5.0))
    # columns that are not turned stay whatever stands beside them
    y = torch.randn(1, 3, 128, device="cuda")
    y[0, 0, 100], y[0, 0, 101] = float("inf"), float("nan")
    for n_rot, neox in ((64, True), (64, False), (10, True)):
        kv4.append4(y.view(1, 384), k, v, pos[:1], slot[:1], q[:1], heads=1, inv_freq=freqs(n_rot), n_rot=n_rot, neox=neox)
        assert torch.equal(q[0, 0, 64:].nan_to_num(nan=5.0, posinf=6.0), y[0, 0, 64:].nan_to_num(nan=5.0, posinf=6.0))


def test_rows_without_a_token():
    """Rows whose position or slot the cache does not have leave cache, queries and results as they are, in every call that takes rows."""
    k, v = filled(2, 2, 70, 64)
    before = [t.clone() for c in (k, v) for t in (c.codes, c.scale)]
    pos, slot = ints(-1, 70, 3, 5, 2 ** 31 - 1, 9), ints(0, 1, -1, 2, 0, 1)
    qkv = torch.randn(6, 8 * 64, device="cuda")
    prep = dict(heads=4, inv_freq=freqs(64), n_rot=64)
    q, out, rows = torch.full((6, 4, 64), 3.0, device="cuda"), torch.full((6, 256), 3.0, device="cuda"), [torch.full((6, 2, 64), 3.0, device="cuda", dtype=F16) for _ in range(2)]
    kv4.append4(qkv, k, v, pos, slot, q, **prep)
    kv4.read4(k, v, pos, slot, *rows)
    assert (q[:5] == 3).all() and all((r[:5] == 3).all() for r in rows) and not (q[5] == 3).any()
    for f in (lambda: kv4.attn_decode4(q, k, v, pos, slot, out, scale=0.1), lambda: kv4.attn_step4(qkv, k, v, pos, slot, out, scale=0.1, **prep)):
        f()
        assert (out[:5] == 3).all() and not (out[5] == 3).any()
        out.fill_(3)
    for c, codes, scale in ((k, *before[:2]), (v, *before[2:])):
        codes[1, :, 9], scale[1, :, 9] = c.codes[1, :, 9], c.scale[1, :, 9]
        assert torch.equal(c.codes, codes) and torch.equal(c.scale, scale)
    kv4.attn_decode4(q[:5], k, v, pos[:5], slot[:5], out[:5], scale=0.1)
    kv4.attn_decode4(q[:0], k, v, pos[:0], slot[:0], out[:0], scale=0.1)
    kv4.append4(qkv[:0], k, v, pos[:0], slot[:0], q[:0], **prep)
    kv4.read4(k, v, pos[:0], slot[:0], rows[0][:0], rows[1][:0])
    assert (out == 3).all()


# ---- single tokens ----------------------------------------------------------------------------------------------------------------
def check_decode(q, k, v, pos, slot, out, **mask):
    kv4.attn_decode4(q, k, v, pos, slot, out, **mask)
    for i, (p, s) in enumerate(zip(pos.tolist(), slot.tolist())):
        want, err = O.attend(q[i:i + 1], values(k, s, p + 1), values(v, s, p + 1), torch.tensor([p]), **mask)
        O.assert_near(out[i:i + 1], want, err)


@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 64), (4, 2, 64), (7, 1, 128), (32, 4, 128), (16, 16, 64), (20, 1, 64), (48, 3, 128), (9, 1, 128)])
@pytest.mark.parametrize("window,softcap,sinks", [(0, 0.0, False), (33, 0.0, True), (0, 5.0, False), (1, 0.0, False), (200, 20.0, True)])
def test_single_tokens(heads, kv_heads, dim, window, softcap, sinks):
    lengths = [1, 2, 31, 33, 128, 129, 300, 1000]
    k, v = filled(len(lengths) + 1, kv_heads, 1009, dim, heads)
    g = gen(dim + window)
    q = torch.randn(len(lengths), heads, dim, device="cuda", generator=g)
    pos, slot = ints(*[n - 1 for n in lengths]), ints(*range(len(lengths), 0, -1))
    s = torch.randn(heads, device="cuda", generator=g) * 3 if sinks else None
    buf = torch.zeros(len(lengths), heads * dim + 5, device="cuda", dtype=B16)
    check_decode(q.to(F16) if window else q, k, v, pos, slot, buf[:, :heads * dim], scale=1.5 / dim ** 0.5, window=window, softcap=softcap, sinks=s)
    assert not buf[:, heads * dim:].any()


@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0])
def test_single_tokens_of_other_scales(scale):
    """fp32 results; with scores of zero the mean of the keys, whose only errors are roundings."""
    k, v = filled(3, 2, 700, 128, 5)
    q = torch.randn(3, 4, 128, device="cuda", generator=gen(8)) * (0.2 if scale == 3.0 else 1)
    check_decode(q, k, v, ints(699, 0, 350), ints(1, 0, 2), torch.zeros(3, 512, device="cuda"), scale=scale)


def test_more_sequences_than_a_warp_has_lanes():
    n = 75
    k, v = filled(n, 2, 400, 64, 3)
    q = torch.randn(n, 6, 64, device="cuda", generator=gen(1))
    pos = torch.randint(0, 400, (n,), device="cuda", generator=gen(2)).int()
    pos[::7] = -1
    slot = torch.randperm(n, device="cuda", generator=gen(3)).int()
    out = torch.full((n, 384), 3.0, device="cuda")
    kv4.attn_decode4(q, k, v, pos, slot, out, scale=0.2, window=150)
    assert (out[::7] == 3).all()
    for i in range(n):
        if pos[i] >= 0:
            p, s = int(pos[i]), int(slot[i])
            O.assert_near(out[i:i + 1], *O.attend(q[i:i + 1], values(k, s, p + 1), values(v, s, p + 1), torch.tensor([p]), scale=0.2, window=150))


@pytest.mark.parametrize("order", ["growing", "falling", "one"])
def test_scores_that_move_the_reference(order):
    """Scores that grow along the sequence by 2^30 and more, fall, or stand out once."""
    n, dim = 1500, 64
    k, v = filled(1, 1, n, dim, 2, spread=0.0)
    size = torch.linspace(0.01, 8, n, device="cuda") if order == "growing" else torch.linspace(8, 0.01, n, device="cuda") if order == "falling" else torch.where(torch.arange(n, device="cuda") == 777, 20.0, 0.1)
    x = torch.randn(1, 1, n, dim, device="cuda", generator=gen(4)) * 0.02
    x[..., 0] = size
    k = kv4.Cache4(*kv4.encode4(x))
    q = torch.zeros(1, 3, dim, device="cuda")
    q[0, :, 0] = torch.tensor([4.0, -4.0, 1.0])
    check_decode(q, k, v, ints(n - 1), ints(0), torch.zeros(1, 3 * dim, device="cuda"), scale=1.0)
    p = kv4.portions4([(0, 1, 0, n - 1)], 3, k)
    out = torch.zeros(1, 3 * dim, device="cuda")
    kv4.attn_prompt4(q, k, v, p, out, scale=1.0)
    O.assert_near(out, *O.attend(q, values(k, 0), values(v, 0), torch.tensor([n - 1]), scale=1.0, wide=O.HALF16))


def test_faint_keys_keep_their_weight():
    """40000 keys of 2^-21 of the heaviest's weight each are a fiftieth of the result, also behind values a thousand times smaller."""
    n, dim, bits = 40000, 64, 21
    x = torch.zeros(1, 1, n, dim, device="cuda")
    x[..., 0] = -7.0
    x[0, 0, 5, 0] = 0.0
    k = kv4.Cache4(*kv4.encode4(x))
    for small in (1.0, 2.0 ** -10):
        y = torch.full((1, 1, n, dim), small, device="cuda")
        y[0, 0, 5] = -small
        v = kv4.Cache4(*kv4.encode4(y))
        q = torch.zeros(1, 1, dim, device="cuda")
        q[0, 0, 0] = 3.0
        scale = bits * 0.6931471805599453 / float(3 * -values(k, 0, 7)[0, 6, 0])
        want, _ = O.attend(q, values(k, 0), values(v, 0), torch.tensor([n - 1]), scale=scale)
        faint = 2 * (n - 1) * 2.0 ** -bits / (1 + (n - 1) * 2.0 ** -bits)
        assert abs(float(want[0, 0]) / small + 1 - faint) < 1e-6
        # weights and queries are f16: both sides of the mean move by 2^-11 each; the scores are the same for all faint keys, off by 2^-11 of 21 bits at most
        out = torch.zeros(1, dim, device="cuda")
        kv4.attn_decode4(q, k, v, ints(n - 1), ints(0), out, scale=scale)
        bound = small * (4 * O.HALF16 + faint * bits * O.HALF16)
        assert (out - want.float()).abs().max() <= bound
        kv4.attn_prompt4(q, k, v, kv4.portions4([(0, 1, 0, n - 1)], 1, k), out, scale=scale)
        assert (out - want.float()).abs().max() <= bound + small * 2 * O.HALF16


def test_values_of_very_different_sizes():
    """A key whose values are 2^24 times another's: relative to the row's own mean size results are as exact as others."""
    n, dim = 600, 128
    g = gen(6)
    k, _ = filled(1, 2, n, dim, 6)
    x = torch.randn(1, 2, n, dim, device="cuda", generator=g) * torch.exp2(torch.randint(-14, 11, (1, 2, n, 1), device="cuda", generator=g).float())
    v = kv4.Cache4(*kv4.encode4(x))
    q = torch.randn(1, 4, dim, device="cuda", generator=g)
    check_decode(q, k, v, ints(n - 1), ints(0), torch.zeros(1, 4 * dim, device="cuda"), scale=0.1)
    zero = kv4.Cache4.empty(1, 2, n, dim)
    out = torch.ones(1, 4 * dim, device="cuda")
    kv4.attn_decode4(q, k, zero, ints(n - 1), ints(0), out, scale=0.1)
    assert not out.any()


@pytest.mark.parametrize("heads,kv_heads,dim,n_rot,neox,norm", [(4, 2, 64, 64, True, False), (32, 8, 128, 128, False, True), (20, 2, 128, 64, True, True), (1, 1, 64, 10, True, False), (16, 16, 64, 0, True, True)])
def test_step_is_append_and_attention(heads, kv_heads, dim, n_rot, neox, norm):
    """The bytes that append4 makes, and attention of the queries that it makes."""
    g, lengths = gen(heads), [1, 7, 128, 129, 500]
    n = len(lengths)
    qkv = torch.randn(n, (heads + 2 * kv_heads) * dim + 1, device="cuda", generator=g)[:, 1:]
    w = [1 + 0.3 * torch.randn(dim, device="cuda", generator=g) for _ in range(2)] if norm else (None, None)
    pos, slot = ints(*[m - 1 for m in lengths]), ints(*range(n - 1, -1, -1))
    prep = dict(heads=heads, inv_freq=freqs(n_rot), n_rot=n_rot, neox=neox, mscale=1.1, q_norm=w[0], k_norm=w[1], eps=1e-6)
    mask = dict(scale=1.2 / dim ** 0.5, window=130, sinks=torch.randn(heads, device="cuda", generator=g))
    a, b = filled(n, kv_heads, 505, dim, 9), filled(n, kv_heads, 505, dim, 9)
    for c in a + b:           # what stood in the rows before does not matter
        c.scale[slot.long(), :, pos.long()] = float("nan")
    q = torch.empty(n, heads, dim, device="cuda", dtype=F16)
    kv4.append4(qkv, *a, pos, slot, q, **prep)
    one, other = torch.zeros(n, heads * dim, device="cuda"), torch.zeros(n, heads * dim, device="cuda")
    kv4.attn_decode4(q, *a, pos, slot, one, **mask)
    kv4.attn_step4(qkv, *b, pos, slot, other, **prep, **mask)
    assert torch.equal(one, other) and all(torch.equal(x.codes, y.codes) and torch.equal(x.scale, y.scale) for x, y in zip(a, b))
    for i, (p, s) in enumerate(zip(pos.tolist(), slot.tolist())):
        O.assert_near(one[i:i + 1], *O.attend(q[i:i + 1], values(a[0], s, p + 1), values(a[1], s, p + 1), torch.tensor([p]), **mask))


# ---- prompts ----------------------------------------------------------------------------------------------------------------------
def check_prompt(q, k, v, parts, out, tail=True, **mask):
    """Over a cache, or over 16-bit tensors [slots, G, positions, D]."""
    heads, cached = q.shape[1], isinstance(k, kv4.Cache4)
    p = kv4.portions4(parts, heads, k, window=mask.get("window", 0))
    before = out[p.rows:].clone()
    launches = (kv4.attn_prompt4 if cached else kv4.attn_packed)(q, k, v, p, out, **mask)
    assert launches == (2 if p.parts else 1)
    for row, n, s, pos, *more in parts:
        base = more[0] if more else 0
        keys, vals = ((O.held(c.codes[s, :, base:base + pos + n], c.scale[s, :, base:base + pos + n]) if cached else c[s, :, base:base + pos + n].double()) for c in (k, v))
        wide = O.HALF16 if cached else 0.0
        want, err = O.attend(q[row:row + n], keys, vals, torch.arange(pos, pos + n), wide=wide + (O.HALFB if not cached and k.dtype == B16 else 0), **mask)
        if not cached and k.dtype == B16:       # weights are bf16 numbers
            err = err + 2 * O.HALFB * O.attend(q[row:row + n], keys, vals.abs(), torch.arange(pos, pos + n), **mask)[0]
        O.assert_near(out[row:row + n], want, err)
    assert torch.equal(out[p.rows:], before) and kv4.status() == 0


@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 64), (4, 2, 64), (7, 1, 128), (32, 4, 128), (16, 16, 64), (40, 2, 128), (130, 2, 64), (128, 1, 128)])
@pytest.mark.parametrize("window,softcap,sinks", [(0, 0.0, False), (33, 0.0, True), (0, 5.0, True), (1, 0.0, False), (300, 0.0, False)])
def test_prompts_over_the_cache(heads, kv_heads, dim, window, softcap, sinks):
    """Portions of one row, of tiles and a row more, beginnings and ends in the middle of a tile of keys."""
    k, v = filled(5, kv_heads, 700, dim, heads)
    g, parts, at = gen(window + dim), [], 0
    for n, slot, pos in ((1, 4, 0), (1, 0, 640), (130, 2, 0), (65, 3, 127), (3, 1, 697)):
        parts.append((at, n, slot, pos))
        at += n
    q = torch.randn(at + 2, heads, dim, device="cuda", generator=g)
    s = torch.randn(heads, device="cuda", generator=g) * 3 if sinks else None
    out = torch.full((at + 2, heads * dim + 8), 3.0, device="cuda", dtype=B16)
    check_prompt(q.to(F16) if window else q, k, v, parts, out[:, :heads * dim], scale=1.5 / dim ** 0.5, window=window, softcap=softcap, sinks=s)
    assert (out[:, heads * dim:] == 3).all()


@pytest.mark.parametrize("rows,pos,scale", [(1, 5000, 0.1), (17, 4500, 0.1), (64, 4990, -0.1), (200, 3000, 0.0), (5, 0, 0.3)])
@pytest.mark.parametrize("q_type,out_type", [(F32, F32), (F16, B16), (B16, F16)])
def test_few_rows_behind_many_keys(rows, pos, scale, q_type, out_type):
    """Keys shared out over CTAs and added up."""
    k, v = filled(2, 2, 5100, 128, rows)
    q = torch.randn(rows, 8, 128, device="cuda", generator=gen(rows)).to(q_type)
    check_prompt(q, k, v, [(0, rows, 1, pos)], torch.zeros(rows, 1024, device="cuda", dtype=out_type), scale=scale)


def test_many_shares_a_cta():
    """More tiles than SMs of all sizes, with and without a second tile of rows, so that CTAs go from share to share."""
    k, v = filled(9, 16, 1300, 64, 1)
    g, parts, at = gen(1), [], 0
    for i in range(40):
        n = (1, 40, 64, 65, 129, 200, 3)[i % 7]
        parts.append((at, n, i % 9, (i * 97) % (1300 - n)))
        at += n
    q = torch.randn(at, 32, 64, device="cuda", generator=g)
    check_prompt(q, k, v, parts, torch.zeros(at, 2048, device="cuda", dtype=B16), scale=0.2)
    check_prompt(q.to(F16), k, v, parts, torch.zeros(at, 2048, device="cuda", dtype=B16), scale=0.2, window=70)
    x = [torch.randn(1, 16, 1300, 64, device="cuda", generator=g).to(F16) for _ in range(2)]
    check_prompt(q.to(F16), *x, [(r, n, 0, p) for r, n, _, p in parts], torch.zeros(at, 2048, device="cuda", dtype=B16), scale=0.2)
    check_prompt(q.to(B16), *x, [(r, n, 0, p) for r, n, _, p in parts], torch.zeros(at, 2048, device="cuda", dtype=B16), scale=-0.2)


@pytest.mark.parametrize("kind,q_type", [(F16, F16), (F16, F32), (B16, B16), (B16, F32), (F16, B16), (B16, F16)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (32, 8, 128), (7, 1, 128), (6, 6, 64)])
def test_packed_rows(kind, q_type, heads, kv_heads, dim):
    """Rows [rows, heads, columns] of sequences one after the other, as they stand in a projection: keys and values of rows with others' columns between them."""
    g, lengths = gen(heads), [1, 2, 127, 128, 129, 257, 64]
    total = sum(lengths)
    buf = torch.randn(total, (heads + 2 * kv_heads) * dim, device="cuda", generator=g)
    q = buf[:, :heads * dim].to(q_type).view(total, heads, dim)
    kv = buf[:, heads * dim:].to(kind).view(total, 2, kv_heads, dim)
    k, v = (kv[:, i].transpose(0, 1)[None] for i in range(2))
    parts, at = [], 0
    for n in lengths:
        parts.append((at, n, 0, 0, at))
        at += n
    for window, sinks in ((0, None), (50, torch.randn(heads, device="cuda", generator=g))):
        check_prompt(q, k, v, parts, torch.zeros(total, heads * dim, device="cuda", dtype=B16), scale=1 / dim ** 0.5, window=window, sinks=sinks)
    # queries out of a wider row, and heads before positions
    wide = torch.zeros(total, heads * dim + 16, device="cuda", dtype=q_type)
    wide[:, :heads * dim] = q.flatten(1)
    check_prompt(wide[:, :heads * dim].view(total, heads, dim), *(x.contiguous() for x in (k, v)), parts, torch.zeros(total, heads * dim, device="cuda"), scale=0.1)


@pytest.mark.parametrize("kind", [F16, B16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_keys_that_a_row_does_not_see(kind, bad):
    """Values and keys that are not finite leave every row that does not see them as it was, bit by bit, and those that see a value without a result."""
    lengths, heads, dim = [100, 90, 300, 5], 4, 64
    total, g = sum(lengths), gen(3)
    q, k, v = (torch.randn(total, n, dim, device="cuda", generator=g).to(kind) for n in (heads, 2, 2))
    parts, at = [], 0
    for n in lengths:
        parts.append((at, n, 0, 0, at))
        at += n
    view = lambda x: x.transpose(0, 1)[None]
    for window in (0, 60):
        p = kv4.portions4(parts, heads, view(k), window=window)
        clean, out = (torch.zeros(total, heads * dim, device="cuda", dtype=B16) for _ in range(2))
        kv4.attn_packed(q, view(k), view(v), p, clean, scale=0.1, window=window)
        for row, what in ((100, "v"), (189, "v"), (190 + 150, "v"), (190 + 299, "v"), (490, "v"), (100, "k"), (190 + 7, "k"), (494, "k")):
            k2, v2 = k.clone(), v.clone()
            (v2 if what == "v" else k2)[row, :, 11] = bad
            kv4.attn_packed(q, view(k2), view(v2), p, out, scale=0.1, window=window)
            first = next(r for r, n, _, _, _ in reversed(parts) if r <= row)
            end = first + lengths[[r for r, *_ in parts].index(first)]
            sees = torch.zeros(total, dtype=torch.bool, device="cuda")
            sees[row:min(end, row + window) if window else end] = True
            assert torch.equal(out[~sees], clean[~sees]), (row, what)
            if what == "v":
                assert not torch.isfinite(out[sees].view(int(sees.sum()), heads, dim)[..., 11].float()).any(), row
    assert kv4.status() == 0


def test_cached_rows_that_no_row_sees():
    """Rows of a cache behind a portion may hold anything."""
    k, v = filled(2, 2, 400, 128, 4)
    q = torch.randn(70, 4, 128, device="cuda", generator=gen(4))
    p = kv4.portions4([(0, 70, 1, 100)], 4, k)
    clean, out = (torch.zeros(70, 512, device="cuda") for _ in range(2))
    kv4.attn_prompt4(q, k, v, p, clean, scale=0.1)
    one = torch.zeros(1, 512, device="cuda")
    kv4.attn_decode4(q[69:], k, v, ints(169), ints(1), one, scale=0.1)
    for c in (k, v):
        c.scale[1, :, 170:] = float("nan")
        c.scale[0] = float("inf")
    kv4.attn_prompt4(q, k, v, p, out, scale=0.1)
    assert torch.equal(out, clean)
    again = torch.zeros(1, 512, device="cuda")
    kv4.attn_decode4(q[69:], k, v, ints(169), ints(1), again, scale=0.1)
    assert torch.equal(one, again)


# ---- together, streams, graphs ----------------------------------------------------------------------------------------------------
def test_a_prompt_and_steps_together():
    """A prompt in two portions, steps behind it, a question of several rows: the cache that results is the one of single rows, attention that of what it holds."""
    heads, kv_heads, dim, n = 8, 2, 128, 180
    g = gen(12)
    qkv = torch.randn(n, (heads + 2 * kv_heads) * dim, device="cuda", generator=g)
    prep = dict(heads=heads, inv_freq=freqs(dim), n_rot=dim)
    k, v = (kv4.Cache4.empty(2, kv_heads, 200, dim) for _ in range(2))
    pos, slot = torch.arange(n, device="cuda", dtype=torch.int32), torch.ones(n, device="cuda", dtype=torch.int32)
    q, out = torch.empty(n, heads, dim, device="cuda", dtype=F16), torch.zeros(n, heads * dim, device="cuda")
    for a, b in ((0, 100), (100, 170), (173, 180)):
        if a == 173:
            for i in range(170, 173):
                kv4.attn_step4(qkv[i:i + 1], k, v, pos[i:i + 1], slot[i:i + 1], out[i:i + 1], scale=0.1, **prep)
        kv4.append4(qkv[a:b], k, v, pos[a:b], slot[a:b], q[a:b], **prep)
        kv4.attn_prompt4(q[a:b], k, v, kv4.portions4([(0, b - a, 1, a)], heads, k), out[a:b], scale=0.1)
    kv4.append4(qkv, *(both := [kv4.Cache4.empty(2, kv_heads, 200, dim) for _ in range(2)]), pos, slot, q, **prep)
    assert all(torch.equal(x.codes[1, :, :n], y.codes[1, :, :n]) and torch.equal(x.scale[1, :, :n], y.scale[1, :, :n]) for x, y in zip((k, v), both))
    want, err = O.attend(q, values(k, 1, n), values(v, 1, n), torch.arange(n), scale=0.1, wide=O.HALF16)
    O.assert_near(out, want, err)


def test_captured_calls_and_other_streams():
    """Two graphs of steps and prompts, replayed in turn and side by side with new inputs; an eager call on a stream of its own."""
    k, v = filled(4, 2, 3000, 64, 7)
    g = gen(7)
    prep = dict(heads=4, inv_freq=freqs(64), n_rot=64)
    made = []
    for i in range(2):
        # each graph has two slots of its own: steps of one slot, or of slots that another call reads, would be in no order
        qkv, pos, slot = torch.randn(2, 512, device="cuda", generator=g), ints(2900 + i, 17), ints(2 * i, 2 * i + 1)
        step, ask = torch.zeros(2, 256, device="cuda"), torch.zeros(40, 256, device="cuda", dtype=B16)
        q = torch.randn(40, 4, 64, device="cuda", generator=g).to(F16)
        p = kv4.portions4([(0, 33, 2 * i + 1, 2800), (33, 7, 2 * i, 50)], 4, k)
        call = lambda qkv=qkv, pos=pos, slot=slot, step=step, ask=ask, q=q, p=p: (kv4.attn_step4(qkv, k, v, pos, slot, step, scale=0.1, **prep), kv4.attn_prompt4(q, k, v, p, ask, scale=0.1))
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        made.append((graph, call, qkv, q, step, ask))
    for turn in range(3):
        for graph, call, qkv, q, step, ask in made:
            qkv.copy_(torch.randn(qkv.shape, device="cuda", generator=g))
            q.copy_(torch.randn(q.shape, device="cuda", generator=g))
        want = []
        for graph, call, _, _, step, ask in made:
            call()
            torch.cuda.synchronize()
            want.append((step.clone(), ask.clone()))
        for _, _, _, _, step, ask in made:
            step.zero_()
            ask.zero_()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in made]
        for s, (graph, call, *_) in zip(streams, made):          # side by side
            with torch.cuda.stream(s):
                graph.replay() if turn < 2 else call()
        torch.cuda.synchronize()
        for (step, ask), (_, _, _, _, a, b) in zip(want, made):
            assert torch.equal(step, a) and torch.equal(ask, b)
    # many of one call's, of the same queries
    outs = [torch.zeros_like(want[0][1]) for _ in range(8)]
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        with torch.cuda.stream(streams[i % 2]):
            kv4.attn_prompt4(made[1][3], k, v, p, o, scale=0.1)
    torch.cuda.synchronize()
    assert all(torch.equal(o, outs[0]) for o in outs) and kv4.status() == 0


def test_threads_side_by_side():
    k, v = filled(2, 2, 900, 128, 5)
    q = torch.randn(20, 8, 128, device="cuda", generator=gen(5))
    pos, slot, p = torch.arange(600, 620, device="cuda", dtype=torch.int32), ints(*[0, 1] * 10), kv4.portions4([(0, 20, 1, 800)], 8, k)
    want = [torch.zeros(20, 1024, device="cuda") for _ in range(2)]
    kv4.attn_decode4(q, k, v, pos, slot, want[0], scale=0.1)
    kv4.attn_prompt4(q, k, v, p, want[1], scale=0.1)
    torch.cuda.synchronize()
    bad = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                out = [torch.zeros(20, 1024, device="cuda") for _ in range(2)]
                kv4.attn_decode4(q, k, v, pos, slot, out[0], scale=0.1)
                kv4.attn_prompt4(q, k, v, p, out[1], scale=0.1)
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(out, want)):
                    bad.append(1)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_rows_beyond_32_bit_offsets():
    """A cache of more than 2^32 bytes and positions whose rows lie beyond them."""
    n_ctx, kv_heads, dim = 9_000_000, 8, 128
    k, v = (kv4.Cache4.empty(1, kv_heads, n_ctx, dim) for _ in range(2))
    heads, rows = 16, 40
    g = gen(2)
    qkv = torch.randn(rows, (heads + 2 * kv_heads) * dim, device="cuda", generator=g)
    pos, slot = torch.arange(n_ctx - rows, n_ctx, device="cuda", dtype=torch.int32), torch.zeros(rows, device="cuda", dtype=torch.int32)
    q = torch.empty(rows, heads, dim, device="cuda", dtype=F16)
    kv4.append4(qkv, k, v, pos, slot, q, heads=heads, inv_freq=freqs(dim), n_rot=dim)
    keys, vals = (O.held(c.codes[0, :, -rows:], c.scale[0, :, -rows:]) for c in (k, v))
    O.assert_held(qkv[:, -kv_heads * dim:].double().view(rows, kv_heads, dim).transpose(0, 1), v.codes[0, :, -rows:], v.scale[0, :, -rows:])
    want, err = O.attend(q, keys, vals, torch.arange(rows), scale=0.1, window=8, wide=O.HALF16)
    one = torch.zeros(1, heads * dim, device="cuda")
    kv4.attn_decode4(q[-1:], k, v, pos[-1:], slot[-1:], one, scale=0.1, window=8)
    O.assert_near(one, want[-1:], err[-1:])
    out = torch.zeros(rows - 8, heads * dim, device="cuda")
    kv4.attn_prompt4(q[8:], k, v, kv4.portions4([(0, rows - 8, 0, n_ctx - rows + 8)], heads, k, window=8), out, scale=0.1, window=8)
    O.assert_near(out, want[8:], err[8:])


# ---- refusals ---------------------------------------------------------------------------------------------------------------------
def test_refusals():
    k, v = filled(2, 2, 50, 64)
    q, qkv, out, pos, slot = torch.zeros(3, 4, 64, device="cuda"), torch.zeros(3, 512, device="cuda"), torch.zeros(3, 256, device="cuda"), ints(1, 2, 3), ints(0, 1, 0)
    f, rows = freqs(64), [torch.zeros(3, 2, 64, device="cuda", dtype=F16) for _ in range(2)]
    other = filled(2, 2, 51, 64)
    append = dict(heads=4, inv_freq=f, n_rot=64)
    bad = [
        (kv4.append4, (qkv.double(), k, v, pos, slot, q), append), (kv4.append4, (qkv[:, :500], k, v, pos, slot, q), append), (kv4.append4, (qkv, k, other[1], pos, slot, q), append),
        (kv4.append4, (qkv, k, v, pos.long(), slot, q), append), (kv4.append4, (qkv, k, v, pos[:2], slot, q), append), (kv4.append4, (qkv, k, v, pos, slot, q[:2]), append), (kv4.append4, (qkv, k, v, pos, slot, q.to(B16)), append),
        (kv4.append4, (qkv, k, v, pos, slot, q), append | dict(heads=3)), (kv4.append4, (qkv, k, v, pos, slot, q), append | dict(n_rot=65)), (kv4.append4, (qkv, k, v, pos, slot, q), append | dict(n_rot=66)),
        (kv4.append4, (qkv, k, v, pos, slot, q), append | dict(inv_freq=f[:5])), (kv4.append4, (qkv, k, v, pos, slot, q), append | dict(inv_freq=f.double())), (kv4.append4, (qkv, k, v, pos, slot, q), append | dict(inv_freq=None)),
        (kv4.append4, (qkv, k, v, pos, slot, q), append | dict(k_norm=f)), (kv4.append4, (qkv.t().contiguous().t(), k, v, pos, slot, q), append), (kv4.append4, (qkv[:1].expand(3, -1), k, v, pos, slot, q), append),
        (kv4.read4, (k, v, pos, slot, rows[0].float(), rows[1]), {}), (kv4.read4, (k, v, pos, slot, rows[0], rows[1][:2]), {}), (kv4.read4, (k, v, pos, slot[:1], *rows), {}),
        (kv4.attn_decode4, (q, k, v, pos, slot, out[:, :200]), dict(scale=1.0)), (kv4.attn_decode4, (q.to(B16), k, v, pos, slot, out), dict(scale=1.0)), (kv4.attn_decode4, (q[:, :3], k, v, pos, slot, out), dict(scale=1.0)),
        (kv4.attn_decode4, (q, k, v, pos, slot, out.to(F16)), dict(scale=1.0)), (kv4.attn_decode4, (q, k, v, pos, slot, out), dict(scale=float("nan"))), (kv4.attn_decode4, (q, k, v, pos, slot, out), dict(scale=float("inf"))),
        (kv4.attn_decode4, (q, k, v, pos, slot, out), dict(scale=1.0, softcap=-1.0)), (kv4.attn_decode4, (q, k, v, pos, slot, out), dict(scale=1.0, softcap=float("inf"))), (kv4.attn_decode4, (q, k, v, pos, slot, out), dict(scale=1.0, window=-1)),
        (kv4.attn_decode4, (q, k, v, pos, slot, out), dict(scale=1.0, sinks=out[0])), (kv4.attn_decode4, (q, k, v, pos, slot, out[:1].expand(3, -1)), dict(scale=1.0)), (kv4.attn_decode4, (q[:, :, :32], k, v, pos, slot, out), dict(scale=1.0)),
        (kv4.attn_step4, (qkv, k, v, pos, slot, out[:2]), append | dict(scale=1.0)), (kv4.attn_step4, (qkv[:, 1:], k, v, pos, slot, out), append | dict(scale=1.0)),
    ]
    p = kv4.portions4([(0, 3, 0, 5)], 4, k)
    x = torch.zeros(2, 2, 50, 64, device="cuda", dtype=F16)
    px = kv4.portions4([(0, 3, 0, 5)], 4, x)
    bad += [
        (kv4.attn_prompt4, (q[:2], k, v, p, out[:2]), dict(scale=1.0)), (kv4.attn_prompt4, (q, *other, p, out), dict(scale=1.0)), (kv4.attn_prompt4, (q, k, v, p, out), dict(scale=1.0, window=3)),
        (kv4.attn_prompt4, (q[:, :2], k, v, p, out), dict(scale=1.0)), (kv4.attn_prompt4, (q.double(), k, v, p, out), dict(scale=1.0)), (kv4.attn_prompt4, (q, k, v, p, out.double()), dict(scale=1.0)),
        (kv4.attn_prompt4, (q.transpose(0, 1), k, v, p, out), dict(scale=1.0)), (kv4.attn_prompt4, (q, k, v, p, torch.zeros(3, 257, device="cuda")[:, 1:]), dict(scale=1.0)), (kv4.attn_prompt4, (q, k, v, p, torch.zeros(3, 257, device="cuda")[:, :256]), dict(scale=1.0)),
        (kv4.attn_packed, (q, x, x[:1], px, out), dict(scale=1.0)), (kv4.attn_packed, (q, x.float(), x.float(), px, out), dict(scale=1.0)), (kv4.attn_packed, (q, x, x.to(B16), px, out), dict(scale=1.0)),
        (kv4.attn_packed, (q, x[:, :, :49], x[:, :, :49], px, out), dict(scale=1.0)), (kv4.attn_packed, (q, x[:, :1].expand(2, 2, 50, 64), x, px, out), dict(scale=1.0)),
        (kv4.attn_packed, (q, torch.zeros(2, 2, 50, 68, device="cuda", dtype=F16)[..., :64], x, px, out), dict(scale=1.0)), (kv4.attn_packed, (q, torch.zeros(2, 2, 50, 128, device="cuda", dtype=F16)[..., ::2], x, px, out), dict(scale=1.0)),
        (kv4.attn_packed, (q, torch.zeros(2 * 2 * 50 * 64 + 1, device="cuda", dtype=F16)[1:].view(2, 2, 50, 64), x, px, out), dict(scale=1.0)),
    ]
    before = [t.clone() for t in (q, out, k.codes, v.codes)]
    for f, args, kw in bad:
        with pytest.raises(ValueError, match=f.__name__):
            f(*args, **kw)
    with pytest.raises(TypeError):
        kv4.attn_decode4([1], k, v, pos, slot, out, scale=1.0)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, (q, out, k.codes, v.codes)))


def test_lists_that_changed_after_they_were_made():
    """Tiles and sums that reach beyond the queries, the cache or the partial results are left out, and the rows of the others are what they were; lists of other lengths are refused."""
    k, v = filled(3, 2, 3000, 64)
    q, one = torch.randn(150, 8, 64, device="cuda", generator=gen(5)).to(F16), kv4.Portions4.__match_args__
    x = [torch.randn(3, 2, 3000, 64, device="cuda", generator=gen(6)).to(F16) for _ in range(2)]
    p = kv4.portions4([(0, 70, 1, 0), (70, 70, 2, 2900)], 8, k)      # the second one's keys are shared out
    assert p.parts > 1 and len(p.merges)
    change = lambda **kw: kv4.Portions4(**({n: getattr(p, n) for n in one} | kw))
    first = (p.tiles[:, 0] < 70).nonzero().view(-1)
    for call, kv in ((kv4.attn_prompt4, (k, v)), (kv4.attn_packed, x)):
        good = torch.full((150, 512), 5.0, device="cuda")
        call(q, *kv, p, good, scale=0.1)
        for column, worth in ((0, -1), (0, 145), (0, 2 ** 31 - 1), (1, 0), (1, -5), (1, 257), (1, 2 ** 31 - 1), (2, 3), (2, -1), (3, -1), (3, 2999), (3, 2 ** 31 - 1), (4, -1), (4, 2950), (4, 2 ** 31 - 1), (5, -1), (5, 30), (6, 0),
                              (6, 2 ** 31 - 1), (7, p.parts), (7, 2 ** 31 - 1), (8, 2), (8, -1)):
            tiles, out = p.tiles.clone(), torch.full((150, 512), 5.0, device="cuda")
            tiles[first, column] = worth
            call(q, *kv, change(tiles=tiles), out, scale=0.1)
            assert (out[:70] == 5).all() and torch.equal(out[70:], good[70:]), (column, worth)
        for column, worth in ((0, -1), (0, 149), (2, -1), (2, p.parts), (2, 2 ** 31 - 1), (3, 0), (3, p.parts + 1), (3, 2 ** 31 - 1), (4, 2), (4, -1)):
            merges, out = p.merges.clone(), torch.full((150, 512), 5.0, device="cuda")
            merges[:, column] = worth
            call(q, *kv, change(merges=merges), out, scale=0.1)
            split = torch.zeros(150, dtype=torch.bool, device="cuda")
            for row, rows in p.merges[:, :2].tolist():
                split[row:row + rows] = True
            assert (out[split] == 5).all() and torch.equal(out[~split], good[~split]), (column, worth)
        for starts in (p.starts - 5, p.starts + len(p.tiles), p.starts * 0 - 2 ** 31, p.starts * 0 + 2 ** 31 - 1, p.starts.flip(0)):
            out = torch.full((150, 512), 5.0, device="cuda")
            call(q, *kv, change(starts=starts.contiguous()), out, scale=0.1)
            assert (out[140:] == 5).all()
        for wrong in (dict(tiles=p.tiles[:3]), dict(tiles=p.tiles.long()), dict(tiles=p.tiles[:, :8].contiguous()), dict(starts=p.starts[:1]), dict(merges=p.merges.float())):
            with pytest.raises(ValueError, match=call.__name__):
                call(q, *kv, change(**wrong), good, scale=0.1)
    torch.cuda.synchronize()
    assert kv4.status() == 0


def test_results_far_apart():
    """Rows of results up to 2^36 bytes from the first, and not beyond."""
    k, v = filled(1, 1, 40, 64)
    q, p = torch.randn(9, 1, 64, device="cuda", generator=gen(7)), kv4.portions4([(0, 9, 0, 20)], 1, k)
    want = torch.zeros(9, 64, device="cuda")
    kv4.attn_prompt4(q, k, v, p, want, scale=0.2)
    step = 2 ** 31 - 4
    far = torch.empty(8 * step + 64, device="cuda")
    kv4.attn_prompt4(q[:8], k, v, kv4.portions4([(0, 8, 0, 20)], 1, k), far.as_strided((8, 64), (step, 1)), scale=0.2)
    assert torch.equal(far.as_strided((8, 64), (step, 1)), want[:8])
    with pytest.raises(ValueError, match="apart"):
        kv4.attn_prompt4(q, k, v, p, far.as_strided((9, 64), (step, 1)), scale=0.2)
