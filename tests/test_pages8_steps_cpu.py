"""Host side of steps whose portions differ: what is read out together."""
import numpy as np
import pytest
import torch

from ollama_b200.ops import pages8 as P


def test_groups_of_pages():
    """Portions in order, as many as fit, tables of pages within the group; one slot's pages always do."""
    table = torch.zeros(5, 20, dtype=torch.int32)
    parts = [(0, 130, 1, 700), (130, 3, 0, 0), (133, 600, 4, 600), (733, 1, 2, 1200), (734, 65, 3, 0)]
    whole = P.portions8(parts, table)
    assert whole.groups == (((0, 0, 0), (10, 17, 54)),) and [s[2] for s in whole.sizes] == [0] * 5
    p = P.portions8(parts, table, together=22)
    # pages seen: 13, 1, 19, 19, 2 -> 14 | 19 | 21
    assert [b[2] - a[2] for a, b in p.groups] == [14, 19, 21] and [s[2] for s in p.sizes] == [0, 0, 1, 2, 2]
    assert [(s[0], s[1]) for s in p.sizes] == [(s[0], s[1]) for s in whole.sizes]
    assert [b[0] - a[0] for a, b in p.groups] == [3, 5, 2] and [b[1] - a[1] for a, b in p.groups] == [4, 10, 3]
    for one, other in ((p.segs, whole.segs), (p.tiles, whole.tiles), (p.half_tiles, whole.half_tiles), (p.pages, whole.pages)):
        assert torch.equal(one, other)
    pages = p.pages.numpy()
    for a, b in p.groups:
        own = pages[a[2]:b[2]]
        assert len(own) <= 22
        for i in sorted(set(p.tiles[a[0]:b[0], 2].tolist())):
            slot = parts[i][2]
            for block in own[own[:, 0] == slot][:, 1]:
                assert own[p.table[i, block]].tolist()[:2] == [slot, block]
    # less than a slot's pages is not asked for
    assert [s[2] for s in P.portions8(parts, table, together=1).sizes] == [0, 0, 1, 2, 3]
    assert max(b[2] - a[2] for a, b in P.portions8(parts, table, together=1).groups) <= 20
    assert np.array_equal(P.portions8(parts[:1], table, together=1).table.numpy(), P.portions8(parts[:1], table).table.numpy())


def test_calls_and_kernels_of_other_sources_are_refused(monkeypatch):
    """The module is the one of these sources, this Python and this torch; it takes a kernel library with the same argument blocks alone."""
    from ollama_b200.kernels import build as B
    from ollama_b200.ops.cuda import lib
    path, text = B.calls_path(), B._text
    for name in ("pages8_args.h", "pages8_call.cpp"):
        with monkeypatch.context() as m:
            m.setattr(B, "_text", lambda *p: text(*p) + (b" " if p[-1] == name else b""))
            assert B.calls_path() != path and (B._layout_flag() != f"-DPAGES8_LAYOUT=0x{_layout(lib()):016x}ull") == (name == "pages8_args.h")
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "1.0")
        assert B.calls_path() != path
    assert B._layout_flag() == f"-DPAGES8_LAYOUT=0x{_layout(lib()):016x}ull"
    P.load()
    m = P._module()
    for wrong in (0, _layout(lib()) + 1):
        with pytest.raises(RuntimeError, match="pages8_args.h"):
            m.bind(1, 2, 3, 4, ValueError, wrong)
    P._bind(m)


def _layout(library):
    import ctypes
    library.b2_pages8_layout.restype = ctypes.c_ulonglong
    return library.b2_pages8_layout()


def test_a_part_of_the_library_comes_with_its_calls(monkeypatch, tmp_path):
    """What a first start compiles for stack models has the module of calls too."""
    from ollama_b200.kernels import build as B
    built = []
    monkeypatch.setattr(B, "_compile", lambda srcs, lib, *a: built.append(lib))
    monkeypatch.setattr(B, "build_calls", lambda *a: built.append("calls"))
    B.build_group("stack")
    assert built[-1] == "calls" and len(built) == 2


def test_calls_that_lack_an_argument():
    """Named in the error; `n_ctx`, which nothing follows from, may be left out."""
    k, v = P.Pages8.empty(2, 1, 64, device="cpu"), P.Pages8.empty(2, 1, 64, device="cpu")
    x, i = torch.zeros(1, 192), torch.zeros(1, dtype=torch.int32)
    a = dict(heads=1, dim=64, vdim=64, q_norm=None, k_norm=None, eps=1e-5, freqs=None, n_rot=0, scale=1.0)
    with pytest.raises(ValueError, match="cpu"):
        P.attn_decode8(x, k, v, i, i, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, 64), **a)
    for name in ("heads", "dim", "vdim", "eps", "n_rot", "scale"):
        with pytest.raises(TypeError, match=name):
            P.attn_decode8(x, k, v, i, i, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, 64), **{n: a[n] for n in a if n != name})


def test_threads_that_need_the_calls_at_once(monkeypatch):
    """One of them builds and binds, the others wait for it."""
    import threading
    import time
    made, calls = [], ("append8", "read8", "attn_decode8", "_attn_prompt8")
    P.load()
    module = P._module()
    for name in calls:
        monkeypatch.delitem(vars(P), name)

    def slow():
        made.append(threading.get_ident())
        time.sleep(0.05)
        return module
    monkeypatch.setattr(P, "_calls", slow)
    got = []
    threads = [threading.Thread(target=lambda i=i: got.append(getattr(P, calls[i % 4]))) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 1 and len(got) == 8
