"""The 4-bit cache's host side: codes in tensor operations, how prompts are dealt out, what calls refuse."""
import itertools
import threading

import pytest
import torch

import kv4_oracle as O
from ollama_b200.ops import kv4


@pytest.mark.parametrize("dim", [64, 128])
def test_codes_of_rows(dim):
    g = torch.Generator().manual_seed(dim)
    x = torch.randn(7, 3, dim, generator=g) * torch.exp2(torch.randint(-30, 16, (7, 3, 1), generator=g).float())
    codes, scale = kv4.encode4(x)
    assert codes.shape == (7, 3, dim // 2) and scale.shape == (7, 3, dim // 32)
    O.assert_held(x.double(), codes, scale)
    assert torch.equal(kv4.decode4(codes, scale).double(), O.held(codes, scale))
    again, d = kv4.encode4(kv4.decode4(codes, scale))           # what is held stays, where its scale is a normal number
    normal = (scale.abs() > 2.0 ** -13)[..., None].expand(*scale.shape, 32).flatten(-2)
    assert torch.equal(kv4.decode4(again, d)[normal], kv4.decode4(codes, scale)[normal])


def test_values_that_are_special():
    x = torch.zeros(6, 64)
    x[1, 3], x[1, 40] = float("inf"), -float("inf")
    x[2, :5] = float("nan")
    x[2, 5] = 2.0
    x[3], x[3, 9] = 1e-9, 70000.0
    x[4, 0], x[4, 1] = 3.0, -3.0
    x[5] = 2.0 ** -24
    y = kv4.decode4(*kv4.encode4(x))
    assert torch.isfinite(y).all() and not y[0].any()
    assert y[1, 3] == 65504 and y[1, 40] == -65504 and y[2, 5] == 2.0 and not y[2, :5].any() and y[3, 9] == 65504
    assert y[4, 1] == -3.0 and y[4, 0] == 3.0 * 7 / 8 and not y[5].any()
    assert torch.equal(y.double(), O.rounded(x))


def covered(p, parts, heads, kv_heads, window):
    """Each share's key tiles, once for each KV head and tile of rows; those that the rows see, and no others."""
    group, step = heads // kv_heads, 2 * (128 // (heads // kv_heads))
    ctas = len(p.starts) - 1
    order = [[i, *range(p.starts[i], p.starts[i + 1])] for i in range(ctas)]
    assert sorted(itertools.chain(*order)) == list(range(len(p.tiles))) and p.starts[0] == ctas
    seen = {}
    for t in p.tiles.tolist():
        row, rows, slot, pos, base, lo, hi, part, kvh = t[:9]
        assert hi > lo and rows <= step
        seen.setdefault((row, kvh), []).append((lo, hi, part, rows, slot, pos, base))
    want = {}
    for row, n, slot, pos, *more in parts:
        for r in range(0, n, step):
            m = min(step, n - r)
            first = max(0, pos + r - window + 1) if window else 0
            for kvh in range(kv_heads):
                want[row + r, kvh] = (m, slot, pos + r, more[0] if more else 0, first // 128, (pos + r + m - 1) // 128 + 1)
    assert seen.keys() == want.keys()
    merges = {(m[0], m[4]): m for m in p.merges.tolist()}
    parts_used = []
    for key, shares in seen.items():
        m, slot, pos, base, lo, hi = want[key]
        shares.sort()
        assert all(s[3:] == (m, slot, pos, base) for s in shares)
        assert [s[0] for s in shares] == [lo, *[s[1] for s in shares[:-1]]] and shares[-1][1] == hi
        if len(shares) == 1:
            assert shares[0][2] == -1 and key not in merges
        else:
            row, rows, first, n, kvh = merges[key][:5]
            assert rows == m and n == len(shares) and sorted(s[2] for s in shares) == list(range(first, first + n))
            parts_used += [s[2] for s in shares]
    assert sorted(parts_used) == list(range(p.parts)) and len(merges) == sum(len(s) > 1 for s in seen.values())


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 2), (32, 8), (7, 1), (40, 2), (128, 1)])
@pytest.mark.parametrize("window", [0, 1, 129, 3000])
def test_prompts_are_dealt_out_whole(heads, kv_heads, window):
    k = torch.empty(5, kv_heads, 9000, 64, dtype=torch.float16)
    for parts in ([(0, 1, 4, 0)], [(0, 7, 0, 901)], [(0, 64, 2, 8900)], [(0, 300, 1, 0), (300, 1, 0, 8999), (301, 130, 1, 77), (431, 5, 3, 3)],
                  [(0, 40, 0, 0, 0), (40, 700, 0, 0, 40), (740, 1, 0, 0, 740)], [(i, 1, i % 5, 37 * i) for i in range(200)], [(0, 2048, 0, 6144)]):
        p = kv4.portions4(parts, heads, k, window=window)
        assert p.rows == parts[-1][0] + parts[-1][1] and p.group == heads // kv_heads and p.cache == (5, kv_heads, 9000, 64)
        covered(p, parts, heads, kv_heads, window)


def test_shares_are_even():
    """Where tiles are cut, no CTA has much more than the others; few keys are not cut."""
    k = torch.empty(1, 8, 60000, 128, dtype=torch.float16)
    for parts in ([(0, 64, 0, 30000)], [(0, 2048, 0, 6144)], [(0, 5, 0, 59000)]):
        p = kv4.portions4(parts, 32, k)
        size = (p.tiles[:, 6] - p.tiles[:, 5]).tolist()
        load = [size[i] + sum(size[p.starts[i]:p.starts[i + 1]]) for i in range(len(p.starts) - 1)]
        assert p.parts and max(load) <= 1.2 * sum(load) / 148 + 6
    assert not kv4.portions4([(0, 300, 0, 0)], 32, k).parts


@pytest.mark.parametrize("parts", [[], [(0, 0, 0, 0)], [(1, 2, 0, 0)], [(0, 2, 0, 0), (3, 1, 0, 0)], [(0, 2, 3, 0)], [(0, 2, -1, 0)], [(0, 2, 0, -1)], [(0, 2, 0, 99)], [(0, 2, 0, 0, 99)], [(0, 2, 0, 0, -1)]])
def test_portions_that_do_not_fit(parts):
    with pytest.raises(ValueError, match="portions4"):
        kv4.portions4(parts, 4, torch.empty(3, 2, 100, 64, dtype=torch.float16))


def test_heads_that_do_not_fit():
    k = torch.empty(3, 2, 100, 64, dtype=torch.float16)
    for heads, window in ((0, 0), (3, 0), (4, -1), (258, 0)):
        with pytest.raises(ValueError, match="portions4"):
            kv4.portions4([(0, 2, 0, 0)], heads, k, window=window)


def test_caches_that_are_none():
    kv4.Cache4.empty(1, 1, 5, 64, device="cpu")
    c, s = torch.zeros(2, 1, 5, 32, dtype=torch.uint8), torch.zeros(2, 1, 5, 2, dtype=torch.float16)
    for codes, scale in ((c[0], s), (c.char(), s), (c, s[:1]), (c, s.float()), (c.transpose(0, 1), s), (c[:, :, :, :16].contiguous(), s[..., :1].contiguous()), (c[:, :, :0], s[:, :, :0])):
        with pytest.raises(ValueError, match="Cache4"):
            kv4.Cache4(codes, scale)
    with pytest.raises(ValueError, match="Cache4"):
        kv4.Cache4.empty(1, 1, 5, 96, device="cpu")


def test_calls_lack_a_gpu_or_an_argument():
    k = kv4.Cache4.empty(1, 1, 8, 64, device="cpu")
    x, i, o = torch.zeros(1, 192), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 64)
    q = x[:, :64].view(1, 1, 64)
    p = kv4.portions4([(0, 1, 0, 0)], 1, k)
    calls = {"append4": ((x, k, k, i, i), dict(heads=1, inv_freq=None, n_rot=0)), "read4": ((k, k, i, i, o, o), {}), "attn_decode4": ((q, k, k, i, i, o), dict(scale=1.0)),
             "attn_step4": ((x, k, k, i, i, o), dict(heads=1, inv_freq=None, n_rot=0, scale=1.0)), "attn_prompt4": ((q, k, k, p, o), dict(scale=1.0)), "attn_packed": ((q, q, q, p, o), dict(scale=1.0))}
    assert set(calls) == set(kv4.CALLS)
    for name, (args, kw) in calls.items():
        call = getattr(kv4, name)
        with pytest.raises(ValueError, match="cpu"):
            call(*args, **kw)
        for n in kw:
            if n != "inv_freq":
                with pytest.raises(TypeError, match=n):
                    call(*args, **{m: v for m, v in kw.items() if m != n})
        with pytest.raises(TypeError):
            call(*args, **kw, other=1)


def test_calls_of_other_argument_blocks(monkeypatch):
    from ollama_b200.kernels import build as B
    path, flag, text = B.calls_path("kv4"), B._layout_flag("kv4"), B._text
    for name, other in (("kv4_args.h", True), ("kv4_call.cpp", False), ("call_args.h", False)):
        with monkeypatch.context() as m:
            m.setattr(B, "_text", lambda *p: text(*p) + (b" " if p[-1] == name else b""))
            assert B.calls_path("kv4") != path and (B._layout_flag("kv4") != flag) == other
    kv4.load()
    m = kv4._module()
    with pytest.raises(RuntimeError, match="kv4_args.h"):
        m.bind(1, 2, 3, 4, 5, ValueError, 0)
    kv4._bind(m)


def test_threads_that_need_the_calls_at_once(monkeypatch):
    kv4.load()
    for name in (*kv4.CALLS, "_plan"):
        monkeypatch.delitem(vars(kv4), name)
    made, module = [], kv4._module()
    monkeypatch.setattr(kv4, "_module", lambda: (made.append(1), module)[1])
    threads = [threading.Thread(target=lambda n=n: getattr(kv4, n)) for n in kv4.CALLS * 2]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 1 and all(n in vars(kv4) for n in kv4.CALLS)


def test_scheduler_counts_four_bits(monkeypatch):
    from types import SimpleNamespace

    from ollama_b200.server import sched
    kv = {"general.architecture": "llama", "llama.block_count": 4, "llama.attention.head_count": 8, "llama.attention.head_count_kv": 2, "llama.embedding_length": 1024}
    model = SimpleNamespace(size=1000, kv=lambda: kv)
    need = {}
    for t in ("f16", "q8_0", "int4"):
        monkeypatch.setenv("OLLAMA_KV_CACHE_TYPE", t)
        need[t] = sched.predict_memory(model, 1000, 2) - 1000
    values = 2 * 4 * 2 * 128 * 1000 * 2
    assert need["f16"] == 2 * values and need["int4"] == values * 9 // 16
    # more than one GPU takes: its group keeps int8
    assert sched.predict_memory(model, 1000, 2, free=1000) >= need["q8_0"]
    kv["llama.attention.key_length"] = 96          # no 4-bit cache
    assert sched.predict_memory(model, 1000, 2) - 1000 == int(2 * 4 * 2 * 96 * 1000 * 2 * (1 + 2 / 32))
