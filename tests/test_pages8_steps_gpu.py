"""The 8-bit paged cache in steps whose portions differ: the memory that calls take, rows that are not there, keys of little weight, and geometries beside those of
test_pages8_gpu.py."""
import math

import pytest
import torch

import pages8_oracle as O
from test_pages8_gpu import Setup, compare, i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def library():
    from ollama_b200.ops import cuda as K
    K.need("stack")
    yield
    assert K.gemm_status() == 0


def numbers(s, seed=1):
    """Every page of the cache holds numbers, in a unit in which they are about one."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    for c in (s.k, s.v):
        c.codes.copy_(torch.randint(0, 256, c.codes.shape, generator=g, device="cuda", dtype=torch.uint8) & 0xb7)       # up to 2^-1
        c.unit.fill_(4.0)


def peak(f):
    """Bytes that a call holds at its most beyond what was held before."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    f()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before


def portions_of(lens, at):
    out, row = [], 0
    for slot, (n, p) in enumerate(zip(lens, at)):
        out.append((row, n, slot, p))
        row += n
    return out


def check_rows_of(s, q, out, row, n, slot, pos, scale):
    """``n`` rows of a portion from its first one on, against 64 bits."""
    k, v = s.values(s.k, slot, pos + n), s.values(s.v, slot, pos + n)
    want, moved = O.attend(q[row:row + n].double(), k, v, O.visible(torch.arange(pos, pos + n), pos + n), scale)
    compare(out[row:row + n].view(n, s.H, s.vdim), want, moved, v.abs().max())


def test_memory_follows_the_rows():
    """A long portion beside single tokens: partial results of the row tiles that there are, not of the longest portion's for each."""
    s = Setup(H=32, G=8, dim=128, norm="", n_rot=0, slots=64, n_ctx=2900)
    numbers(s)
    parts = portions_of([2048] + [1] * 63, [0] + [2790 + i for i in range(63)])
    q = torch.randn(2048 + 63, 32, 128, device="cuda")
    out, plan = torch.zeros(len(q), 32 * 128, device="cuda"), s.P.portions8(parts, s.table)
    # tiles of 128 rows: 64 + 63 of each of the 8 KV heads, and one a CTA that fits the GPU; 130 floats a row
    tiles = 8 * (64 + 63) + torch.cuda.get_device_properties(0).multi_processor_count
    assert peak(lambda: s.P.attn_prompt8(q, s.k, s.v, plan, s.table, out, vdim=128, scale=0.2)) <= tiles * 128 * 130 * 4 + (1 << 20)
    for row, n, slot, pos in (parts[1], parts[7], parts[-1], (0, 40, 0, 0)):
        check_rows_of(s, q, out, row, n, slot, pos, 0.2)
    at = torch.arange(2000, 2048)
    k, v = s.values(s.k, 0, 2048), s.values(s.v, 0, 2048)
    want, moved = O.attend(q[at].double(), k, v, O.visible(at, 2048), 0.2)
    compare(out[at].view(48, 32, 128), want, moved, v.abs().max())


def test_long_tables_beside_many_portions():
    """Counts of (keys, row tiles) that fit 32 bits, where the longest portion's tiles times all portions' do not."""
    s = Setup(H=32, G=8, dim=128, norm="", n_rot=0, slots=256, n_ctx=128)
    numbers(s)
    table = torch.full((256, 20000), -1, dtype=torch.int32, device="cuda")
    table[:, :2] = s.table
    table[0, :32] = torch.arange(32, dtype=torch.int32)
    s.table = table
    parts = portions_of([2048] + [1] * 255, [0] + [i % 128 for i in range(255)])
    q = torch.randn(2048 + 255, 32, 128, device="cuda")
    out, plan = torch.zeros(len(q), 32 * 128, device="cuda"), s.P.portions8(parts, table)
    s.P.attn_prompt8(q, s.k, s.v, plan, table, out, vdim=128, scale=0.2)
    s.table = table[:, :64]
    for row, n, slot, pos in (parts[1], parts[100], parts[-1], (0, 40, 0, 0)):
        check_rows_of(s, q, out, row, n, slot, pos, 0.2)


@pytest.mark.parametrize("n", [257, 300])
def test_more_portions_than_a_launch_takes(n):
    """The largest batch of portions is not the first."""
    s = Setup(H=8, G=2, dim=64, norm="", n_rot=0, slots=n, n_ctx=128)
    numbers(s)
    lens = [1 + i % 3 for i in range(256)] + [40] * (n - 256)
    parts = portions_of(lens, [(7 * i) % (128 - m + 1) for i, m in enumerate(lens)])
    q = torch.randn(sum(lens), 8, 64, device="cuda")
    for rows in (n, 200):          # tiles of 128 and 16 rows, and of 8
        out = torch.zeros(len(q), 512, device="cuda")
        some = parts[:rows]
        s.P.attn_prompt8(q, s.k, s.v, s.P.portions8(some, s.table), s.table, out, vdim=64, scale=0.3)
        for row, m, slot, pos in [*some[::17], *some[-3:]]:
            check_rows_of(s, q, out, row, m, slot, pos, 0.3)
        end = some[-1][0] + some[-1][1]
        assert (out[end:] == 0).all()


def test_queries_of_rows_that_are_not_there():
    """Rows whose slot or position the table does not have: their queries are left as they are, as those of rows that hold no token."""
    for append in (True, False):
        s = Setup(H=4, G=2, dim=64, norm="", slots=3, n_ctx=130)          # three pages a slot: positions up to 191
        slots, pos = [0, 7, -1, 3, 1, 2, 2, 1], [5, 5, 6, 0, 191, 192, 2 ** 31 - 1, -1]
        x = s.rnd(8, s.ld)
        q = torch.full((8, 4, 64), 9.0, device="cuda")
        before = s.k.codes.clone()
        s.P.append8(x.cuda(), s.k, s.v, s.table, q, positions=i32(pos), slots=i32(slots), append=append, **s.prep())
        there = [0, 4]
        want = s.split(x, torch.tensor(pos))[0][there]
        assert (q[there].double().cpu() - want).abs().max() <= 2.0 ** -20 * want.abs().max()
        assert (q[[1, 2, 3, 5, 6, 7]] == 9.0).all()
        touched = {int(s.table[0, 0]), int(s.table[1, 2])} if append else set()
        rest = [p for p in range(len(before)) if p not in touched]
        assert torch.equal(s.k.codes[rest], before[rest])


@pytest.mark.parametrize("diff", [False, True])
def test_pages_are_read_out_in_passes(diff):
    """What is held in 16 bits at a time is bounded, and the results are those of one pass."""
    from ollama_b200.ops import rows as R
    s = Setup(H=32, G=8, dim=64 if diff else 128, vdim=128, norm="", n_rot=0, maps=2 if diff else 1, slots=3, n_ctx=1300)
    numbers(s)
    parts = portions_of([600, 500, 640], [600, 700, 640])
    q, outs = torch.randn(1740, 32, 128, device="cuda"), []
    how = dict(diff=R.DiffHeads(0.3, 0.8, 1e-5, 1)) if diff else {}
    for together, pages in ((1024, 58), (1, 20)):
        out, plan = torch.zeros(1740, 16 * 128 if diff else 32 * 128, device="cuda", dtype=torch.bfloat16), s.P.portions8(parts, s.table, together=together)
        # nothing but the pages, keys and values in 16 bits
        assert peak(lambda: s.P.attn_prompt8(q, s.k, s.v, plan, s.table, out, vdim=128, scale=0.2, **how)) <= pages * 2 * 8 * 64 * 128 * 2 + (1 << 16)
        outs.append(out)
    assert torch.equal(*outs) and (outs[0] != 0).any(1).all()


def test_prompts_without_memory_to_read_pages_out(monkeypatch):
    """The other forms take the step where an allocation fails."""
    s = Setup(H=8, G=2, dim=64, norm="", n_rot=0, slots=2, n_ctx=700)
    numbers(s)
    parts = portions_of([300, 280], [300, 0])
    q, plan = torch.randn(580, 8, 64, device="cuda"), s.P.portions8(parts, s.table)
    out = torch.zeros(580, 512, device="cuda", dtype=torch.bfloat16)

    def full(*a, **k):
        raise torch.OutOfMemoryError("no memory")
    with monkeypatch.context() as m:
        m.setattr(torch, "empty", full)
        s.P.attn_prompt8(q, s.k, s.v, plan, s.table, out, vdim=64, scale=0.2)
    for row, n, slot, pos in parts:
        check_rows_of(s, q, out, row, n, slot, pos, 0.2)


def test_other_threads_run_while_a_call_launches(tmp_path):
    """A launch that has to wait holds up its own thread alone.  The entry points are one that sleeps, and launches nothing."""
    import ctypes
    import subprocess
    import threading
    import time
    from ollama_b200.ops import pages8 as P
    src = tmp_path / "wait.c"
    src.write_text("#include <unistd.h>\nint wait_a_little(void) { usleep(300000); return 0; }\n")
    subprocess.run(["g++", "-x", "c", "-shared", "-fPIC", "-o", str(tmp_path / "wait.so"), str(src)], check=True)
    wait = ctypes.CDLL(str(tmp_path / "wait.so")).wait_a_little
    s = Setup(H=4, G=2, dim=64)
    x, q, out, prep = s.rnd(2, s.ld).cuda(), torch.empty(2, 4, 64, device="cuda"), torch.empty(2, 256, device="cuda"), s.prep()
    plan, pages, wide = P.portions8([(0, 2, 0, 0)], s.table), i32([[0, 0, 64, 0]]), [torch.zeros(1, 2, 64, 64, device="cuda", dtype=torch.float16) for _ in range(2)]
    P.load()
    m, at, stop, ticks = P._module(), ctypes.cast(wait, ctypes.c_void_p).value, threading.Event(), []
    layout = P.lib().b2_pages8_layout()

    def count():
        while not stop.wait(0.002):
            ticks.append(time.perf_counter())
    t = threading.Thread(target=count)
    m.bind(at, at, at, at, ValueError, layout)
    t.start()
    try:
        for call in (lambda: P.append8(x, s.k, s.v, s.table, q, portions=plan, **prep), lambda: P.read8(s.k, s.v, pages, s.table, *wide),
                     lambda: P.attn_decode8(x, s.k, s.v, i32([0, 0]), i32([0, 1]), s.table, out, n_ctx=64, scale=0.1, **prep),
                     lambda: P.attn_prompt8(q, s.k, s.v, plan, s.table, out, vdim=64, scale=0.1)):
            before = len(ticks)
            call()
            assert len(ticks) - before > 20          # of some 150
    finally:
        stop.set()
        t.join()
        P._bind(m)


def test_calls_from_several_threads():
    """Each on a stream and a cache of its own."""
    import threading
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                s = Setup(H=8, G=2, dim=64, slots=2, n_ctx=400, seed=i)
                numbers(s, i)
                q = torch.randn(300, 8, 64, device="cuda")
                for _ in range(20):
                    for n, dtype in ((300, torch.bfloat16), (60, torch.float32), (2, torch.float32)):
                        out = torch.zeros(n, 512, device="cuda", dtype=dtype)
                        s.P.attn_prompt8(q[:n], s.k, s.v, s.P.portions8([(0, n, 1, 40)], s.table), s.table, out, vdim=64, scale=0.2)
                        check_rows_of(s, q, out, 0, n, 1, 40, 0.2)
        except BaseException as e:
            wrong.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


def test_pages_that_are_read_out_keep_no_tensor_maps():
    """The maps of caches that stay are not pushed out by buffers of single calls."""
    from ollama_b200.ops.cuda import lib
    s = Setup(H=8, G=2, dim=64, norm="", n_rot=0, slots=1, n_ctx=2000)
    numbers(s)
    q, before = torch.randn(300, 8, 64, device="cuda"), lib().b2_attn_prefill_kept_maps()
    for pos in (0, 100, 700, 1500):
        out, plan = torch.zeros(300, 512, device="cuda", dtype=torch.bfloat16), s.P.portions8([(0, 300, 0, pos)], s.table)
        pages = plan.groups[0][1][2]
        assert peak(lambda: s.P.attn_prompt8(q, s.k, s.v, plan, s.table, out, vdim=64, scale=0.2)) >= 2 * pages * 2 * 64 * 64 * 2          # read out first
        check_rows_of(s, q, out, 0, 300, 0, pos, 0.2)
    assert lib().b2_attn_prefill_kept_maps() == before


@pytest.mark.parametrize("form", ["rows", "tiles", "read out"])
def test_faint_keys_of_long_sequences(form):
    """Eight keys that share nearly all of the weight, one for each warp and one or more for each group, and 100000 of e^-17.5 (2^-25.2) each, whose values are what the result is.
    Queries, keys and values are exact in 16 and in 8 bits, so that only the weights' rounding to f16 is left: of 2^-19.2 at least, whose half step is 2^-25, so 2^-5.8 of them."""
    keys, slots, n, dtype = 100000, *{"rows": (256, 1, torch.float32), "tiles": (148, 40, torch.float32), "read out": (1, 5120, torch.bfloat16)}[form]
    s = Setup(H=4, G=1, dim=64, norm="", n_rot=0, slots=1, n_ctx=keys)
    at = s.table[0].long()
    k, v = torch.zeros(len(at) * 64, 64), torch.ones(len(at) * 64, 64)
    k[:, 0] = 0.5
    k[:256:32, 0], v[:256:32] = 18.0, 0.0
    for c, x in ((s.k, k), (s.v, v)):
        c.unit.fill_(1.0)
        c.codes.zero_()
        c.codes[at] = x.view(len(at), 1, 64, 64).to(torch.float8_e4m3fn).view(torch.uint8).cuda()
    table = s.table.expand(slots, -1).contiguous()          # pages that nothing is appended to may be in several slots
    q = torch.zeros(slots * n, 4, 64, device="cuda")
    q[..., 0] = 1.0
    out = torch.zeros(slots * n, 256, device="cuda", dtype=dtype)
    s.P.attn_prompt8(q, s.k, s.v, s.P.portions8(portions_of([n] * slots, [keys - n] * slots), table), table, out, vdim=64, scale=1.0)
    faint = torch.arange(keys - n - 7, keys - 7, dtype=torch.float64, device="cuda").repeat(slots)[:, None] * math.exp(-17.5)
    want = faint / (8 + faint)
    off = (out.double() - want).abs() / want
    assert off.max() <= 2.0 ** -5.8 + 2.0 ** -10 + (2.0 ** -8 if dtype == torch.bfloat16 else 0), float(off.max())


@pytest.mark.parametrize("append", [True, False])
def test_launches_are_counted(append):
    """What the engine adds to its count is what a capture of the same calls holds."""
    import ctypes

    from ollama_b200.engine.mixers import attend8
    from ollama_b200.ops import rows as O8
    for lens, dtype, together in (([3, 2], torch.bfloat16, 1024), ([300, 260], torch.bfloat16, 1024), ([300, 260], torch.bfloat16, 1), ([2] * 300, torch.float32, 1024)):
        s = Setup(H=8, G=2, dim=64, norm="", slots=len(lens), n_ctx=320, seed=71)
        numbers(s)
        x = s.rnd(sum(lens), s.ld).cuda()
        plan, prep = s.P.portions8(portions_of(lens, [10] * len(lens)), s.table, together=together), s.prep()
        out, q = torch.zeros(len(x), 512, device="cuda", dtype=dtype), torch.zeros(len(x), 512, device="cuda")
        m = type("Meta", (), {"portions": lambda self, table, **how: plan})()
        be = type("Engine", (), {"cache": type("Cache", (), {"table": s.table})()})()
        step = lambda: attend8(be, m, False, x, s.k, s.v, out, 64, lambda *a: q, O8.NO_DIFF, dict(prep, append=append), dict(scale=0.1))  # noqa: E731
        step()
        g = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(g):
            n = step()
        nodes = ctypes.c_size_t()
        assert ctypes.CDLL("libcudart.so.12").cudaGraphGetNodes(ctypes.c_void_p(g.raw_cuda_graph()), None, ctypes.byref(nodes)) == 0
        assert nodes.value == n


def test_units_at_their_borders():
    """448 units are the most that a unit holds: the next larger number takes twice the unit, of one row and of a page's rows, keys and values."""
    top = [448.0 * 2.0 ** e for e in (-15, -3, 0, 6, 7)]
    above = [math.nextafter(t, math.inf) for t in top]
    up = [torch.nextafter(torch.tensor(t), torch.tensor(math.inf)).item() for t in top]
    assert all(u > a for u, a in zip(up, above))          # the next 32-bit number
    want = [2.0 ** e for e in (-15, -3, 0, 6, 7)] + [2.0 ** e for e in (-14, -2, 1, 7, 7)]
    m = [*top, *up]
    s = Setup(H=1, G=1, dim=64, norm="", n_rot=0, slots=10, n_ctx=64)
    x = torch.zeros(10, s.ld)
    for i, t in enumerate(m):
        x[i, s.nq + 3 * i], x[i, s.v_off + 5] = -t, t
    q = torch.empty(10, 1, 64, device="cuda")
    s.P.append8(x.cuda(), s.k, s.v, s.table, q, positions=i32([0] * 10), slots=i32(list(range(10))), **s.prep())
    p = s.table[:, 0].long()
    assert s.k.unit[p, 0].tolist() == want and s.v.unit[p, 0].tolist() == want
    assert s.k.numbers[p, 0, 0].float().abs().amax(1).tolist() == [448.0] * 5 + [224.0] * 4 + [448.0]
    t = Setup(H=1, G=1, dim=64, norm="", n_rot=0, slots=10, n_ctx=64)
    y, q = torch.zeros(30, t.ld), torch.empty(30, 1, 64, device="cuda")
    y[1::3] = x
    t.P.append8(y.cuda(), t.k, t.v, t.table, q, portions=t.P.portions8([(3 * i, 3, i, 0) for i in range(10)], t.table), **t.prep())
    p = t.table[:, 0].long()
    assert t.k.unit[p, 0].tolist() == want and t.v.unit[p, 0].tolist() == want


@pytest.mark.parametrize("G", [3, 5, 6, 7, 8, 9, 12])
def test_norms_over_rows_of_any_number_of_heads(G):
    """A page's KV heads exchange their parts of a norm where they are up to eight, and read the row where they are more."""
    s = Setup(H=2 * G, G=G, dim=32, norm="row", slots=2, n_ctx=200, seed=G)
    x, q = s.rnd(170, s.ld), torch.empty(170, 2 * G, 64, device="cuda")
    parts = [(0, 130, 1, 20), (130, 40, 0, 0)]
    s.P.append8(x.cuda(), s.k, s.v, s.table, q, portions=s.P.portions8(parts, s.table), **s.prep())
    pos = torch.cat([torch.arange(p, p + n) for _, n, _, p in parts])
    qx, kx, vx = s.split(x, pos)
    assert (q[..., :32].double().cpu() - qx).abs().max() <= 2.0 ** -20 * qx.abs().max() and (q[..., 32:] == 0).all()
    for row, n, slot, p in parts:
        s.check_rows(s.k, 32, slot, p, kx[row:row + n])
        s.check_rows(s.v, 32, slot, p, vx[row:row + n])


@pytest.mark.parametrize("gate", ["element", "head"])
def test_difference_of_maps_with_a_gate(gate):
    from ollama_b200.ops import rows as R
    heads, kv, dim, vdim, lam, factor, eps, scale = 8, 2, 32, 64, 0.37, 0.8, 1e-5, 0.2
    s = Setup(H=heads, G=kv, dim=dim, vdim=vdim, norm="", maps=2, slots=1, n_ctx=500, seed=61)
    diff, at = R.DiffHeads(lam, factor, eps, 1), 0
    for n in (3, 60, 300, 1):
        x, gv = s.rnd(n, s.ld), s.rnd(n, heads // 2 * vdim).cuda()
        out = torch.zeros(n, heads // 2 * vdim, device="cuda", dtype=torch.bfloat16)
        if n > 1:
            q, plan = torch.empty(n, heads, s.hd, device="cuda"), s.P.portions8([(0, n, 0, at)], s.table)
            s.P.append8(x.cuda(), s.k, s.v, s.table, q, portions=plan, **s.prep())
            s.P.attn_prompt8(q, s.k, s.v, plan, s.table, out, vdim=vdim, scale=scale, gate=R.head_gate(gv, gate), diff=diff)
        else:
            s.P.attn_decode8(x.cuda(), s.k, s.v, i32([at]), i32([0]), s.table, out, n_ctx=500, scale=scale, gate=R.head_gate(gv, gate), diff=diff, **s.prep())
        pos = torch.arange(at, at + n)
        qx = s.split(x, pos)[0].cuda()
        k, v = s.values(s.k, 0, at + n), s.values(s.v, 0, at + n)
        o = [O.attend(qx[:, m::2], k[..., m * dim:(m + 1) * dim], v[..., :vdim], O.visible(pos, at + n), scale) for m in range(2)]
        d = o[0][0] - lam * o[1][0]
        rms = (d.square().mean(-1, keepdim=True) + eps).sqrt()
        near = (O.tolerance(o[0][0], o[0][1], v.abs().max(), torch.float32) + lam * O.tolerance(o[1][0], o[1][1], v.abs().max(), torch.float32)).amax(-1, keepdim=True)
        f = torch.sigmoid(gv.double()).view(n, heads // 2, vdim) if gate == "element" else torch.sigmoid(gv[:, :heads // 2].double())[..., None]
        want = d / rms * factor * f
        # the norm divides the difference's error and moves by as much itself; the gate's exponential and quotient are off by some 2^-21
        assert ((out.double().view(n, heads // 2, vdim) - want).abs() <= 2 * factor * f * near / rms + want.abs() * (2.0 ** -8 + 2.0 ** -20)).all()
        at += n


def test_products_behind_the_attention_are_as_fast_as_elsewhere():
    """The attention leaves SMs with most of their L1 as shared memory; the products that stream a model's weights behind it take their own split.  Graphs of both, of the attention
    alone and of the products alone, in turn on one GPU: a fourth more without, 2 % with it."""
    from ollama_b200.ops import rows as R
    s = Setup(H=16, G=4, dim=128, norm="", slots=1, n_ctx=6400)
    numbers(s)
    n, k, each, w = 5120, 2048, 12, []                     # 12 x 21 MB, more than L2 holds; one wave of CTAs each, all of whose loads are under way at once
    for _ in range(each):
        w.append(torch.randn(n, k, device="cuda").bfloat16())
    x, y = torch.randn(1, k, device="cuda").bfloat16(), torch.zeros(1, n, device="cuda")
    qkv, out, a, prep = s.rnd(1, s.ld).cuda(), torch.zeros(1, 2048, device="cuda"), (i32([6000]), i32([0]), s.table), s.prep()
    graphs = []
    for attention, product in ((True, True), (True, False), (False, True)):
        def run():
            for i in range(each):
                if attention:
                    s.P.attn_decode8(qkv, s.k, s.v, *a, out, scale=0.1, pdl=True, **prep)
                if product:
                    for j in range(4):
                        R.gemv([R.seg(w[(4 * i + j) % each], n, y)], k, x, 1, False, pdl=True)
        run()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run()
        graphs.append(g)
    times = ([], [], [])
    for i in range(25):
        for g, t in zip(graphs, times):
            b, e = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            b.record()
            g.replay()
            e.record()
            torch.cuda.synchronize()
            if i >= 5:
                t.append(b.elapsed_time(e))
    both, attention, product = (sorted(t)[len(t) // 2] for t in times)
    assert both - attention < 1.12 * product, (both, attention, product)


def test_portions_that_were_not_made_as_such_are_refused():
    """What the calls take from them without looking at their rows: types, shapes, how many there are."""
    import dataclasses
    s = Setup(H=4, G=2, dim=64)
    q, out = torch.zeros(5, 4, 64, device="cuda"), torch.zeros(5, 256, device="cuda")
    x, prep = s.rnd(5, s.ld).cuda(), s.prep()
    good = s.P.portions8([(0, 2, 0, 0), (2, 3, 1, 5)], s.table)
    before = s.k.codes.clone()
    segs = (good.segs.long(), good.segs[:1].expand(2, 4), good.segs.t().contiguous(), good.segs.view(-1), good.segs.float(), good.segs.cpu(), torch.zeros(9, dtype=torch.int32, device="cuda")[1:].view(2, 4))
    for bad in (dataclasses.replace(good, segs=t) for t in segs):
        with pytest.raises(ValueError):
            s.P.append8(x, s.k, s.v, s.table, q, portions=bad, **prep)
        with pytest.raises(ValueError):
            s.P.attn_prompt8(q, s.k, s.v, bad, s.table, out, vdim=64, scale=0.1)
    for bad in (dict(sizes=list(good.sizes)), dict(sizes=good.sizes[:1]), dict(sizes=tuple(x[:2] for x in good.sizes)), dict(sizes=tuple(list(x) for x in good.sizes)), dict(masks=[0, 0, 0]),
                dict(masks=(0, 0)), dict(table=good.table[0]), dict(table=good.table[:, :2])):
        with pytest.raises(ValueError):
            s.P.attn_prompt8(q, s.k, s.v, dataclasses.replace(good, **bad), s.table, out, vdim=64, scale=0.1)
    for bad in (None, 3, (0, 1)):
        with pytest.raises((AttributeError, TypeError, ValueError)):
            s.P.attn_prompt8(q, s.k, s.v, bad, s.table, out, vdim=64, scale=0.1)
    assert torch.equal(s.k.codes, before) and (out == 0).all()


def test_pages_that_have_changed_are_refused():
    """Tensors of a cache that were changed in place after it was made, objects that only look like one, and codes off 16-byte boundaries."""
    from types import SimpleNamespace
    s = Setup(H=4, G=2, dim=64)
    P, x, q, prep = s.P, s.rnd(1, s.ld).cuda(), torch.zeros(1, 4, 64, device="cuda"), s.prep()
    one, zero = i32([5]), i32([0])

    def calls(k, v, table=s.table):
        yield lambda: P.append8(x, k, v, table, q, positions=one, slots=zero, **prep)
        yield lambda: P.attn_decode8(x, k, v, one, zero, table, torch.zeros(1, 256, device="cuda"), scale=0.1, **prep)
        yield lambda: P.attn_prompt8(q, k, v, P.portions8([(0, 1, 0, 0)], s.table), table, torch.zeros(1, 256, device="cuda"), vdim=64, scale=0.1)
        yield lambda: P.read8(k, v, i32([[0, 0, 64, 0]]), table, *(torch.zeros(1, 2, 64, 64, device="cuda", dtype=torch.float16) for _ in range(2)))
    n = s.k.codes.shape[0]
    short, flat, off = P.Pages8.empty(n, 2, 64), P.Pages8.empty(n, 2, 64), torch.zeros(n * 2 * 64 * 64 + 1, device="cuda", dtype=torch.uint8)[1:].view(n, 2, 64, 64)
    short.unit.resize_(n - 1, 2)
    flat.codes.resize_(n, 2 * 64 * 64)
    bad = [(short, s.v), (s.k, short), (flat, flat), (P.Pages8(off, torch.ones(n, 2, device="cuda")), s.v)]
    bad += [(SimpleNamespace(codes=s.k.codes, unit=u), s.v) for u in (s.k.unit.double(), s.k.unit.cpu(), s.k.unit.t(), s.k.unit[:, :1])]
    bad += [(SimpleNamespace(codes=c, unit=s.k.unit), s.v) for c in (s.k.codes.cpu(), s.k.codes.view(torch.int8), s.k.codes[:, :, :32], s.k.codes.transpose(2, 3))]
    for k, v in bad:
        for call in calls(k, v):
            with pytest.raises(ValueError):
                call()
    for call in calls(s.k, s.v, s.table[:0]):
        with pytest.raises(ValueError):
            call()
