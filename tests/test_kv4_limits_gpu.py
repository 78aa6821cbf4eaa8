"""The 4-bit cache's and packed prompts' attention where keys are cut into parts: sinks that are not finite, rows alone and beside others."""
import pytest
import torch

import kv4_oracle as O
from ollama_b200.ops import kv4
from test_kv4_gpu import filled, gen, ints, values

pytestmark = pytest.mark.gpu
F16 = torch.float16


def sixteen_bit(slots, kv_heads, n_ctx, dim, seed):
    return [torch.randn(slots, kv_heads, n_ctx, dim, device="cuda", generator=gen(seed + i)).to(F16) for i in range(2)]


def assert_sinks(attend):
    """``attend(sinks)`` -> results [rows, 4 heads, columns]: exp(inf) in the denominator leaves nothing, exp(-inf) adds nothing, no number none."""
    inf = float("inf")
    plain, got = attend(None), attend(torch.tensor([inf, -inf, float("nan"), 0.5], device="cuda"))
    assert (got[:, 0] == 0).all() and torch.equal(got[:, 1], plain[:, 1]) and got[:, 2].isnan().all()
    assert ((got[:, 3].abs() < plain[:, 3].abs()) | (plain[:, 3] == 0) & (got[:, 3] == 0)).all()      # (single keys have columns that are held as zeros)


@pytest.mark.parametrize("lengths", [[1], [40], [6000], [70 + 50 * i for i in range(40)]])
def test_infinite_sinks_of_single_tokens(lengths):
    """One part, many of one sequence (eight warps a head add them up), few of each of many (one warp does)."""
    n = len(lengths)
    k, v = filled(n, 1, max(lengths), 64, n)
    q = torch.randn(n, 4, 64, device="cuda", generator=gen(1))

    def attend(sinks):
        out = torch.full((n, 256), 7.0, device="cuda")
        kv4.attn_decode4(q, k, v, ints(*[m - 1 for m in lengths]), ints(*range(n)), out, scale=0.1, sinks=sinks)
        return out.view(n, 4, 64)
    assert_sinks(attend)


@pytest.mark.parametrize("cached", [True, False])
@pytest.mark.parametrize("parts,cut", [([(0, 100, 0, 0)], False), ([(0, 300, 0, 0)], True), ([(0, 5, 0, 5000)], True)])
def test_infinite_sinks_of_prompts(parts, cut, cached):
    """A whole tile, and parts that one warp a row adds up, or eight."""
    k, v = filled(1, 1, 5100, 64, 3) if cached else sixteen_bit(1, 1, 5100, 64, 3)
    rows = parts[-1][0] + parts[-1][1]
    q, p = torch.randn(rows, 4, 64, device="cuda", generator=gen(2)), kv4.portions4(parts, 4, k)
    assert (p.parts > 0) == cut

    def attend(sinks):
        out = torch.full((rows, 256), 7.0, device="cuda")
        (kv4.attn_prompt4 if cached else kv4.attn_packed)(q, k, v, p, out, scale=0.1, sinks=sinks)
        return out.view(rows, 4, 64)
    assert_sinks(attend)
    assert kv4.status() == 0


def assert_same_but_for_roundings(a, b, q, keys, vals, pos, scale):
    """Two results of the same rows whose keys were cut at other places: scores are the same, weights are f16 numbers relative to other references (2^-11 each), sums have another order (2^-18 as in
    kv4_oracle.attend), weights that are subnormals move the mean by 2^-31 of the largest value for each key, and each result is rounded to fp32.  The mean size is taken from exact scores, 5 % are for
    theirs."""
    size = O.attend(q.to(F16), keys, vals.abs(), pos, scale=scale)[0] * 1.05
    off = 2 * (O.HALF16 + 2.0 ** -18) * size + 2 * keys.shape[1] * 2.0 ** -31 * vals.abs().max() + 2 * 2.0 ** -22 * size
    assert torch.isfinite(a).all() and ((a.double() - b.double()).abs() <= off).all(), float(((a.double() - b.double()).abs() / off).max())


def test_a_sequence_alone_and_beside_others():
    """Where a sequence's keys are cut follows from all sequences of a call; its result does but for roundings."""
    lengths = [5000, 300, 4100, 1, 900, 2222, 3333, 128]
    n, scale = len(lengths), 0.1
    k, v = filled(n, 2, 5000, 128, 4)
    q = torch.randn(n, 8, 128, device="cuda", generator=gen(5))
    pos, slot = ints(*[m - 1 for m in lengths]), ints(*range(n))
    out, one = torch.zeros(n, 1024, device="cuda"), torch.zeros(n, 1024, device="cuda")
    kv4.attn_decode4(q, k, v, pos, slot, out, scale=scale)
    for i, m in enumerate(lengths):
        kv4.attn_decode4(q[i:i + 1], k, v, pos[i:i + 1], slot[i:i + 1], one[i:i + 1], scale=scale)
        assert_same_but_for_roundings(out[i:i + 1], one[i:i + 1], q[i:i + 1], values(k, i, m), values(v, i, m), torch.tensor([m - 1]), scale)


@pytest.mark.parametrize("cached", [True, False])
def test_a_portion_alone_and_beside_others(cached):
    """The same of portions: alone their keys are cut at other places than beside others, or not at all."""
    scale, heads = 0.1, 8
    k, v = filled(3, 2, 5100, 128, 6) if cached else sixteen_bit(3, 2, 5100, 128, 6)
    parts = [(0, 7, 1, 5000), (7, 150, 0, 4200), (157, 64, 2, 4990), (221, 1, 0, 40), (222, 300, 1, 0)]
    q = torch.randn(522, heads, 128, device="cuda", generator=gen(6)).to(F16)
    call, p = kv4.attn_prompt4 if cached else kv4.attn_packed, kv4.portions4(parts, heads, k)
    out, cuts = torch.zeros(522, 1024, device="cuda"), {tuple(t[:3]) for t in p.merges[:, [0, 1, 3]].tolist()}
    call(q, k, v, p, out, scale=scale)
    other = 0
    for row, n, s, pos in parts:
        alone = kv4.portions4([(0, n, s, pos)], heads, k)
        other += any((row + r, m, c) not in cuts for r, m, c in alone.merges[:, [0, 1, 3]].tolist())
        one = torch.zeros(n, 1024, device="cuda")
        call(q[row:row + n], k, v, alone, one, scale=scale)
        keys, vals = (values(c, s, pos + n) if cached else c[s, :, :pos + n].double() for c in (k, v))
        assert_same_but_for_roundings(out[row:row + n], one, q[row:row + n], keys, vals, torch.arange(pos, pos + n), scale)
    assert other >= 2 and kv4.status() == 0


@pytest.mark.parametrize("rows", [256, 288])
def test_both_ways_of_adding_up(rows):
    """Sums of more than four parts, of 1024 rows (tiles of 256, four KV heads), which eight warps each add up, and of 2048, which one does."""
    k, v = filled(1, 4, 30100, 64, 7)
    heads = 4
    q, pos = torch.randn(rows, heads, 64, device="cuda", generator=gen(rows)).to(F16), 30000 - rows
    p = kv4.portions4([(0, rows, 0, pos)], heads, k)
    assert p.parts / len(p.merges) > 4
    out = torch.zeros(rows, heads * 64, device="cuda")
    kv4.attn_prompt4(q, k, v, p, out, scale=0.1)
    some = torch.arange(0, rows, 37, device="cuda")
    want, err = O.attend(q[some], values(k, 0, pos + rows), values(v, 0, pos + rows), pos + some, scale=0.1, wide=O.HALF16)
    O.assert_near(out[some], want, err)
    assert kv4.status() == 0
