"""The 8-bit paged cache against its definition in 64 bits: rows appended, pages read back, decode and prompt attention, and all of them as a program runs them."""
import math

import pytest
import torch

import pages8_oracle as O

pytestmark = pytest.mark.gpu
F64 = torch.float64
NAN8 = 0x7f


@pytest.fixture(scope="module", autouse=True)
def library():
    from ollama_b200.ops import cuda as K
    K.need("stack")
    yield
    assert K.gemm_status() == 0


def i32(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


class Setup:
    """A cache of scattered pages for slots 0 .. ``slots`` - 1 and one layer's geometry.  Pages start with NaN in every code and a unit of their own, so that what should
    not be read shows."""

    def __init__(self, H=4, G=2, dim=64, vdim=None, slots=3, n_ctx=300, norm="head", n_rot=None, maps=1, keys_as_values=False, mscale=1.0, seed=0, extra=3, first_page=0):
        from ollama_b200.ops import pages8 as P
        self.P, self.H, self.G, self.dim, self.vdim, self.maps, self.mscale = P, H, G, dim, vdim or dim, maps, mscale
        self.g = torch.Generator().manual_seed(seed)
        self.kdim, self.nq, self.nk = maps * dim, H * dim, G * maps * dim
        self.hd = 64 if max(self.kdim, self.vdim) <= 64 else 128
        n_rot = dim // 2 * 2 if n_rot is None else n_rot
        self.freqs = 700.0 ** (-torch.arange(n_rot // 2, dtype=F64) * 2 / max(n_rot, 1))
        self.f = (self.freqs if n_rot else torch.zeros(1, dtype=F64)).cuda()
        self.n_rot, self.eps, self.head_norm = n_rot, 1e-5, norm == "head"
        n = (dim, dim) if norm == "head" else (self.nq, self.nk)
        self.qn, self.kn = (1 + 0.3 * self.rnd(n[0]), 1 + 0.3 * self.rnd(n[1])) if norm else (None, None)
        self.v_off = self.nq if keys_as_values else self.nq + self.nk
        self.ld = self.nq + self.nk + (0 if keys_as_values else G * self.vdim)
        pages = -(-n_ctx // 64)
        n_pages = first_page + slots * pages + extra
        self.table = (first_page + torch.randperm(slots * pages + extra, generator=self.g)[:slots * pages]).view(slots, pages).to(torch.int32).cuda()
        self.k, self.v = P.Pages8.empty(n_pages, G, self.hd), P.Pages8.empty(n_pages, G, self.hd)
        for c in (self.k, self.v):
            c.codes[first_page:] = NAN8
            c.unit[first_page:] = 2.0 ** -15

    def rnd(self, *s):
        return torch.randn(*s, generator=self.g)

    def prep(self):
        c = lambda t: None if t is None else t.cuda()  # noqa: E731
        self.held = [c(self.qn), c(self.kn)]
        return dict(heads=self.H, dim=self.dim, vdim=self.vdim, q_norm=self.held[0], k_norm=self.held[1], eps=self.eps, freqs=self.f, n_rot=self.n_rot, head_norm=self.head_norm,
                    v_off=self.v_off, mscale=self.mscale, maps=self.maps)

    def split(self, x, pos):
        """(queries, keys, values) of raw rows in 64 bits, as they go into the attention and the cache."""
        x, n = x.double(), len(x)
        q = O.normed(x[:, :self.nq].view(n, self.H, self.dim), self.qn, self.eps, self.head_norm)
        k = O.normed(x[:, self.nq:self.nq + self.nk].view(n, self.G * self.maps, self.dim), self.kn, self.eps, self.head_norm)
        q, k = (O.rotated(t, pos, self.freqs, self.mscale) for t in (q, k))
        return q, k.reshape(n, self.G, self.kdim), x[:, self.v_off:self.v_off + self.G * self.vdim].view(n, self.G, self.vdim)

    def caches(self):
        return O.Cache(torch.nan_to_num(self.k.numbers.float(), nan=0.0).cpu(), self.k.unit.cpu()), O.Cache(torch.nan_to_num(self.v.numbers.float(), nan=0.0).cpu(), self.v.unit.cpu())

    def check_rows(self, c, cols, slot, pos, x):
        """Rows at ``pos`` .. of a slot hold ``x`` within half a step of E4M3 in their page's unit; the rotation's 32 bits move a value by 2^-20 of the row's size at most."""
        num, unit = c.numbers.float().double().cpu(), c.unit.double().cpu()
        at = torch.arange(pos, pos + len(x))
        page = self.table.cpu()[slot, at // 64].long()
        got = num[page, :, at % 64] * unit[page][..., None]
        u = unit[page][..., None]
        tol = torch.maximum(x.abs() * 2.0 ** -4, u * 2.0 ** -10) + x.abs().amax() * 2.0 ** -20
        assert (got[..., :cols] - x).abs().le(tol).all()
        assert (got[..., cols:] == 0).all()

    def values(self, c, slot, n):
        """[kv heads, n, columns] of a slot as the cache has them, in 64 bits, what is no number as zero."""
        x = torch.nan_to_num(c.numbers.float().double(), nan=0.0) * c.unit.double()[..., None, None]
        return x[self.table[slot].long()].transpose(0, 1).reshape(self.G, -1, self.hd)[:, :n]

    def fill(self, slot, n, spread=1.0):
        """Positions 0 .. n - 1 of a slot get random values."""
        from ollama_b200.ops import pages8 as P
        x = self.rnd(n, self.ld) * spread
        q = torch.empty(n, self.H, self.hd, device="cuda")
        P.append8(x.cuda(), self.k, self.v, self.table, q, portions=P.portions8([(0, n, slot, 0)], self.table), **self.prep())


GEOMETRIES = [dict(H=4, G=2, dim=64), dict(H=32, G=8, dim=128, norm="row"), dict(H=6, G=2, dim=48, vdim=40), dict(H=3, G=1, dim=100, vdim=30, norm="row"),
              dict(H=5, G=5, dim=30, vdim=29, n_rot=12), dict(H=2, G=1, dim=128, vdim=64, norm=""), dict(H=8, G=2, dim=24, vdim=50, norm="", maps=2, mscale=1.2),
              dict(H=4, G=4, dim=40, n_rot=0, keys_as_values=True), dict(H=40, G=2, dim=64, vdim=1, norm="row"), dict(H=12, G=3, dim=1, vdim=128, n_rot=0, norm="")]


@pytest.mark.parametrize("geometry", GEOMETRIES)
def test_append_of_portions(geometry):
    s = Setup(slots=4, n_ctx=400, seed=geometry["dim"], **geometry)
    P, kc, vc = s.P, *s.caches()
    held = [0, 0, 0, 0]
    for lens in ([1, 63, 64, 65], [62, 2, 1, 130], [3, 128, 200, 7], [64, 0, 65, 1]):
        parts, at = [], 0
        for slot in (2, 0, 3, 1):
            if lens[slot]:
                parts.append((at, lens[slot], slot, held[slot]))
                at += lens[slot]
        x = s.rnd(at, s.ld) * torch.exp2(3 * s.rnd(at, 1))       # rows of very different sizes: units grow
        q = torch.full((at, s.H, s.hd), 9.0, device="cuda")
        P.append8(x.cuda(), s.k, s.v, s.table, q, portions=P.portions8(parts, s.table), **s.prep())
        pos = torch.cat([torch.arange(p, p + n) for _, n, _, p in parts])
        qx, kx, vx = s.split(x, pos)
        full = torch.zeros(at, s.H, s.hd, dtype=F64)
        for h in range(s.H):
            o = h % s.maps * s.dim
            full[:, h, o:o + s.dim] = qx[:, h]
        assert (q.double().cpu() - full).abs().max() <= 2.0 ** -20 * full.abs().max()
        for row, n, slot, p in parts:
            kc.append(s.table, slot, p, kx[row:row + n])
            vc.append(s.table, slot, p, vx[row:row + n])
            s.check_rows(s.k, s.kdim, slot, p, kx[row:row + n])
            s.check_rows(s.v, s.vdim, slot, p, vx[row:row + n])
            held[slot] += n
    for got, want in ((s.k, kc), (s.v, vc)):
        for slot, n in enumerate(held):
            pages = s.table[slot, :-(-n // 64)].long().cpu()
            assert torch.equal(got.unit.cpu()[pages].double(), want.u[pages])          # random magnitudes are nowhere near a border
            a, b = (t[pages].transpose(0, 1).reshape(s.G, -1, s.hd)[:, :n] for t in (got.numbers.float().double().cpu(), want.n))
            # a value at a border between two numbers may go either way, a step of 1/8 at most
            assert ((a - b).abs() <= b.abs() / 8 + 2.0 ** -9).all() and (a != b).double().mean() < 1e-3
    unused = sorted(set(range(len(s.k.unit))) - {int(p) for slot in range(4) for p in s.table[slot, :-(-held[slot] // 64)]})
    assert (s.k.codes[unused] == NAN8).all() and (s.v.codes[unused] == NAN8).all() and (s.k.unit[unused] == 2.0 ** -15).all()


@pytest.mark.parametrize("geometry", GEOMETRIES)
def test_append_of_single_rows(geometry):
    """One token a sequence, several steps across a page's end; rows without a token, of slots, positions and pages that are not there."""
    s = Setup(slots=3, n_ctx=130, seed=7, **geometry)
    P, kc, vc = s.P, *s.caches()
    s.table[1, 2] = len(s.k.unit) + 5            # a page that is not there
    before = [t.clone() for t in (s.k.codes, s.k.unit, s.v.codes, s.v.unit)]
    for step, (p0, p1, p2) in enumerate([(0, 126, 62), (1, 127, 63), (2, 128, 64), (3, 129, 65)]):
        slots, pos = [2, 1, 0, 0, 7, -1], [p0, p1, p2, -1, 5, 6]
        x = s.rnd(6, s.ld) * 4.0 ** step
        q = torch.full((6, s.H, s.hd), 9.0, device="cuda")
        P.append8(x.cuda(), s.k, s.v, s.table, q, positions=i32(pos), slots=i32(slots), **s.prep())
        qx, kx, vx = s.split(x, torch.tensor(pos))
        assert (q[:3, :, :1].double().cpu()[..., 0] - torch.stack([qx[:3, h, 0] if h % s.maps == 0 else torch.zeros(3, dtype=F64) for h in range(s.H)], 1)).abs().max() <= 1e-4 * qx.abs().max()
        assert (q[3] == 9.0).all()
        for i in range(3):
            if (slots[i], pos[i] // 64) == (1, 2):
                continue
            kc.append(s.table, slots[i], pos[i], kx[i:i + 1])
            vc.append(s.table, slots[i], pos[i], vx[i:i + 1])
    for got, want, was in ((s.k, kc, before[:2]), (s.v, vc, before[2:])):
        touched = [(2, 0, range(0, 4)), (1, 1, range(62, 64)), (0, 0, range(62, 64)), (0, 1, range(0, 2))]
        for slot, b, rows in touched:
            p, rows = int(s.table[slot, b]), list(rows)
            assert torch.equal(got.unit[p].double().cpu(), want.u[p])
            a, w = got.numbers[p][:, rows].float().double().cpu(), want.n[p][:, rows]
            assert ((a - w).abs() <= w.abs() / 8 + 2.0 ** -9).all()
        rest = sorted(set(range(len(got.unit))) - {int(s.table[t, b]) for t, b, _ in touched})
        assert torch.equal(got.codes[rest], was[0][rest]) and torch.equal(got.unit[rest], was[1][rest])


def test_rows_of_one_slot_are_appended_in_order():
    a, b = Setup(H=2, G=2, dim=64, seed=5), Setup(H=2, G=2, dim=64, seed=5)
    x = a.rnd(6, a.ld) * torch.tensor([1.0, 30.0, 0.1, 9.0, 200.0, 3.0])[:, None]
    slots, pos = [1, 0, 1, 1, 0, 1], [62, 3, 63, 64, 3, 65]
    q = torch.empty(6, 2, 64, device="cuda")
    a.P.append8(x.cuda(), a.k, a.v, a.table, q, positions=i32(pos), slots=i32(slots), **a.prep())
    for i in range(6):
        b.P.append8(x[i:i + 1].cuda(), b.k, b.v, b.table, q[:1], positions=i32(pos[i:i + 1]), slots=i32(slots[i:i + 1]), **b.prep())
    for t in ("codes", "unit"):
        assert torch.equal(getattr(a.k, t), getattr(b.k, t)) and torch.equal(getattr(a.v, t), getattr(b.v, t))


def test_append_of_what_is_no_number():
    """NaN stays NaN and does not move the unit; what is too large becomes the largest value; zeros stay zeros."""
    s = Setup(H=2, G=1, dim=64, norm="", n_rot=0)
    x = torch.ones(3, s.ld)
    x[0, s.nq], x[0, s.nq + 1] = math.nan, 3.0
    x[1, s.v_off], x[1, s.v_off + 1] = math.inf, -1e9
    x[2, s.nq:] = 0.0
    q = torch.empty(3, 2, 64, device="cuda")
    s.P.append8(x.cuda(), s.k, s.v, s.table, q, positions=i32([0, 0, 0]), slots=i32([0, 1, 2]), **s.prep())
    p = s.table[:, 0].long()
    k, v = (c.numbers[p, 0, 0].float() * c.unit[p] for c in (s.k, s.v))
    assert k[0, 0].isnan() and k[0, 1] == 3.0 and s.k.unit[p[0], 0] == 2.0 ** -7
    assert v[1, 0] == 57344 and v[1, 1] == -57344 and s.v.unit[p[1], 0] == 2.0 ** 7
    assert (k[2] == 0).all() and (v[2] == 0).all() and s.k.unit[p[2], 0] == 2.0 ** -15


def test_attention_over_what_is_no_number():
    """A key or a value that is no number leaves queries without a result that see it, and no others."""
    for what, dtype in (("k", torch.float32), ("v", torch.float32), ("k", torch.bfloat16), ("v", torch.bfloat16)):
        s = Setup(H=4, G=2, dim=64, norm="", n_rot=0, slots=1, n_ctx=300, seed=3)
        x = s.rnd(200, s.ld)
        x[150, (s.nq if what == "k" else s.v_off) + 64 + 5] = math.nan           # KV head 1
        q, plan = torch.empty(200, 4, 64, device="cuda"), s.P.portions8([(0, 200, 0, 0)], s.table)
        s.P.append8(x.cuda(), s.k, s.v, s.table, q, portions=plan, **s.prep())
        for mask in (dict(), dict(window=20), dict(window=30, keep=4), dict(chunk=64)):
            out = torch.zeros(200, 256, device="cuda", dtype=dtype)
            s.P.attn_prompt8(q, s.k, s.v, s.P.portions8([(0, 200, 0, 0)], s.table, **mask), s.table, out, vdim=64, scale=0.1, **mask)
            sees = O.visible(torch.arange(200), 200, **mask)[:, 150].cuda()
            o = out.view(200, 4, 64)
            assert torch.isfinite(o[:, :2]).all() and torch.isfinite(o[~sees]).all() and o[sees][:, 2:].isnan().any(-1).all()
            for p in (150, 169, 170, 180, 199):                                    # a row appended again: its own key is none only at 150
                y, out1 = x[p:p + 1].cuda(), torch.zeros(1, 256, device="cuda", dtype=dtype)
                s.P.attn_decode8(y, s.k, s.v, i32([p]), i32([0]), s.table, out1, n_ctx=300, scale=0.1, **s.prep(), **mask)
                o1 = out1.view(4, 64)
                assert torch.isfinite(o1[:2]).all() and (o1[2:].isnan().any(-1).all() if sees[p] else torch.isfinite(o1[2:]).all())


@pytest.mark.parametrize("hd,G", [(64, 1), (128, 3)])
def test_read_back(hd, G):
    from ollama_b200.ops import pages8 as P
    g = torch.Generator().manual_seed(3)
    n = 9
    codes = torch.randint(0, 256, (n, G, 64, hd), generator=g, dtype=torch.int32).to(torch.uint8).cuda()
    unit = torch.exp2(torch.randint(-15, 8, (n, G), generator=g).float()).cuda()
    k, v = P.Pages8(codes, unit), P.Pages8(codes.flip(0).contiguous(), unit.flip(0).contiguous())
    table = i32([[4, 2, 8, 99], [0, 1, 3, -1]])
    pages = [(0, 0, 64, 0), (1, 2, 17, 0), (0, 2, 0, 0), (1, 0, 1, 0), (0, 3, 64, 0), (1, 3, 64, 0), (2, 0, 64, 0), (-1, 0, 64, 0), (0, 4, 64, 0), (0, -1, 64, 0), (1, 1, 63, 0)]
    out = [torch.full((len(pages), G, 64, hd), 7.0, device="cuda", dtype=torch.float16) for _ in range(2)]
    P.read8(k, v, i32(pages), table, *out)
    for c, o in zip((k, v), out):
        for i, (t, b, rows, _) in enumerate(pages):
            there = 0 <= t < 2 and 0 <= b < 4 and 0 <= int(table[t, b]) < n
            if there and rows:
                p = int(table[t, b])
                assert torch.equal(torch.nan_to_num(o[i, :, :rows].float(), nan=1e9), torch.nan_to_num(c.numbers[p, :, :rows].float() * c.unit[p][:, None, None], nan=1e9))
            assert (o[i, :, rows if there else 0:] == 0).all()


MASKS = [dict(), dict(window=20, keep=3), dict(window=100, keep=70), dict(window=1, keep=0), dict(window=64), dict(window=1000, keep=9), dict(chunk=37), dict(chunk=128), dict(chunk=1),
         dict(softcap=5.0), dict(window=65, keep=200)]


def compare(got, want, moved, v_max, maps=1):
    err = (got.double() - want).abs()
    tol = O.tolerance(want, moved, v_max, got.dtype)
    assert torch.isfinite(got).all() and (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("geometry", [GEOMETRIES[i] for i in (0, 1, 3, 4, 8)])
def test_decode_attention(geometry, mask):
    lens = [1, 2, 63, 64, 65, 129, 257, 300]
    s = Setup(slots=len(lens), n_ctx=320, seed=11, **geometry)
    for slot, n in enumerate(lens):
        if n > 1:
            s.fill(slot, n - 1)
    order = torch.randperm(len(lens), generator=s.g).tolist()
    slots, pos = order + [0], [lens[i] - 1 for i in order] + [-1]          # the last row holds no token
    x = s.rnd(len(slots), s.ld)
    for gate, dtype in (("", torch.bfloat16), ("element", torch.float32), ("head", torch.bfloat16)):
        from ollama_b200.ops import rows as R
        gv = s.rnd(len(slots), s.H * s.vdim + 3).cuda()
        out = torch.full((len(slots), s.H * s.vdim + 5), 5.0, device="cuda", dtype=dtype)
        m = dict(scale=1.3 / math.sqrt(s.dim), **mask)
        s.P.attn_decode8(x.cuda(), s.k, s.v, i32(pos), i32(slots), s.table, out, n_ctx=320, gate=R.head_gate(gv, gate) if gate else R.NO_GATE, **s.prep(), **m)
        assert (out[-1] == 5).all() and (out[:, s.H * s.vdim:] == 5).all()
        q, kx, vx = s.split(x, torch.tensor(pos))
        for i, slot in enumerate(order):
            s.check_rows(s.k, s.kdim, slot, pos[i], kx[i:i + 1])
            k, v = s.values(s.k, slot, lens[slot]), s.values(s.v, slot, lens[slot])
            softcap = m.get("softcap", 0.0)
            seen = O.visible(torch.tensor([pos[i]]), lens[slot], **{n: mask[n] for n in mask if n != "softcap"})
            want, moved = O.attend(q[i:i + 1].cuda(), k[..., :s.dim], v[..., :s.vdim], seen, m["scale"], softcap)
            f = torch.sigmoid(gv[i].double()) if gate else None
            f = f[:s.H * s.vdim].view(1, s.H, s.vdim) if gate == "element" else f[:s.H].view(1, s.H, 1) if gate else 1.0
            compare(out[i:i + 1, :s.H * s.vdim].view(1, s.H, s.vdim), want * f, moved, v.abs().max())


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("geometry", [GEOMETRIES[i] for i in (0, 1, 3, 4, 8)])
def test_prompt_attention(geometry, mask):
    from ollama_b200.ops import rows as R
    s = Setup(slots=3, n_ctx=700, seed=13, **geometry)
    held = [0, 0, 0]
    for lens in ([5, 1, 64], [200, 2, 129], [1, 17, 63], [130, 300, 1]):
        parts, at = [], 0
        for slot in (1, 2, 0):
            parts.append((at, lens[slot], slot, held[slot]))
            at += lens[slot]
        x, q = s.rnd(at, s.ld), torch.empty(at + 1, s.H, s.hd, device="cuda")
        plan = s.P.portions8(parts, s.table, **{n: mask[n] for n in mask if n != "softcap"})
        s.P.append8(x.cuda(), s.k, s.v, s.table, q[:at], portions=plan, **s.prep())
        gate = ("", "element", "head")[at % 3]
        gv = s.rnd(at + 1, s.H * s.vdim).cuda()
        out = torch.full((at + 1, s.H * s.vdim + 8), 5.0, device="cuda", dtype=torch.bfloat16)
        q[at] = 1.0
        s.P.attn_prompt8(q, s.k, s.v, plan, s.table, out, vdim=s.vdim, scale=1.3 / math.sqrt(s.dim), gate=R.head_gate(gv, gate) if gate else R.NO_GATE, **mask)
        assert (out[at] == 5).all() and (out[:, s.H * s.vdim:] == 5).all()
        for row, n, slot, p in parts:
            held[slot] += n
            pos = torch.arange(p, p + n)
            k, v = s.values(s.k, slot, p + n), s.values(s.v, slot, p + n)
            seen = O.visible(pos, p + n, **{m: mask[m] for m in mask if m != "softcap"})
            want, moved = O.attend(q[row:row + n, :, :s.dim].double(), k[..., :s.dim], v[..., :s.vdim], seen, 1.3 / math.sqrt(s.dim), mask.get("softcap", 0.0))
            f = torch.sigmoid(gv[row:row + n].double()).view(n, s.H, s.vdim) if gate == "element" else torch.sigmoid(gv[row:row + n, :s.H].double())[..., None] if gate else 1.0
            compare(out[row:row + n, :s.H * s.vdim].view(n, s.H, s.vdim), want * f, moved, v.abs().max())


@pytest.mark.parametrize("heads,kv,dim,vdim", [(8, 2, 24, 50), (4, 2, 64, 128), (32, 8, 32, 64)])
def test_differential_attention(heads, kv, dim, vdim):
    """Two maps a head, whose difference is normalised; and queries of a layer that reads another layer's cache."""
    from ollama_b200.ops import rows as R
    s = Setup(H=heads, G=kv, dim=dim, vdim=vdim, norm="", maps=2, slots=2, n_ctx=400, seed=17)
    lam, factor, eps = 0.37, 0.8, 1e-5
    diff, scale = R.DiffHeads(lam, factor, eps, 1), 1.2 / math.sqrt(dim)

    def expect(q, slot, pos, n):
        k, v = s.values(s.k, slot, n), s.values(s.v, slot, n)
        q = q.cuda().double()
        o = []
        for m in range(2):
            r, moved = O.attend(q[:, m::2], k[..., m * dim:(m + 1) * dim], v[..., :vdim], O.visible(pos, n), scale)
            o.append((r, moved))
        d = o[0][0] - lam * o[1][0]
        rms = (d.square().mean(-1, keepdim=True) + eps).sqrt()
        tol = (O.tolerance(o[0][0], o[0][1], v.abs().max(), torch.float32) + lam * O.tolerance(o[1][0], o[1][1], v.abs().max(), torch.float32)).amax(-1, keepdim=True)
        want = d / rms * factor
        return want, 2 * factor * tol / rms + want.abs() * 2.0 ** -8     # the norm divides the difference's error, and moves by as much itself

    for n, p in ((150, 0), (33, 150), (1, 183)):
        x = s.rnd(n, s.ld)
        q = torch.empty(n, heads, s.hd, device="cuda")
        plan = s.P.portions8([(0, n, 1, p)], s.table)
        s.P.append8(x.cuda(), s.k, s.v, s.table, q, portions=plan, **s.prep())
        out = torch.full((n, heads // 2 * vdim + 2), 5.0, device="cuda", dtype=torch.bfloat16)
        s.P.attn_prompt8(q, s.k, s.v, plan, s.table, out, vdim=vdim, scale=scale, diff=diff)
        want, tol = expect(s.split(x, torch.arange(p, p + n))[0], 1, torch.arange(p, p + n), p + n)
        assert ((out[:, :-2].double().view(n, heads // 2, vdim) - want).abs() <= tol).all() and (out[:, -2:] == 5).all()
    x = s.rnd(1, s.ld)
    before = [t.clone() for t in (s.k.codes, s.k.unit, s.v.codes, s.v.unit)]
    out = torch.zeros(1, heads // 2 * vdim, device="cuda")
    s.P.attn_decode8(x[:, :s.nq].contiguous().cuda(), s.k, s.v, i32([100]), i32([1]), s.table, out, n_ctx=200, scale=scale, diff=diff, append=False, **s.prep())
    assert all(torch.equal(a, b) for a, b in zip(before, (s.k.codes, s.k.unit, s.v.codes, s.v.unit)))
    want, tol = expect(s.split(x, torch.tensor([100]))[0], 1, torch.tensor([100]), 101)
    assert ((out.double().view(1, heads // 2, vdim) - want).abs() <= tol).all()


def test_all_in_turn_on_another_stream():
    """A prompt in portions, decode steps beside it, what the cache holds read back; the calls run on a stream of their own."""
    s = Setup(H=8, G=2, dim=128, slots=2, n_ctx=600, seed=23)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    rows = {0: [], 1: []}
    with torch.cuda.stream(st):
        held = [0, 0]
        for lens in ([130, 1], [70, 200], [1, 1], [1, 1], [66, 3], [1, 1]):
            parts = [(0, lens[0], 0, held[0]), (lens[0], lens[1], 1, held[1])]
            x = s.rnd(sum(lens), s.ld)
            for row, n, slot, _ in parts:
                rows[slot].append(x[row:row + n])
            out = torch.empty(len(x), s.H * s.vdim, device="cuda", dtype=torch.bfloat16)
            if sum(lens) == 2:
                s.P.attn_decode8(x.cuda(), s.k, s.v, i32(held), i32([0, 1]), s.table, out, n_ctx=600, scale=0.1, **s.prep())
            else:
                q = torch.empty(len(x), s.H, s.hd, device="cuda")
                plan = s.P.portions8(parts, s.table)
                s.P.append8(x.cuda(), s.k, s.v, s.table, q, portions=plan, **s.prep())
                s.P.attn_prompt8(q, s.k, s.v, plan, s.table, out, vdim=s.vdim, scale=0.1)
            held = [h + n for h, n in zip(held, lens)]
        pages = [(t, b, min(64, held[t] - 64 * b), 0) for t in range(2) for b in range(-(-held[t] // 64))]
        wide = [torch.empty(len(pages), s.G, 64, s.hd, device="cuda", dtype=torch.float16) for _ in range(2)]
        s.P.read8(s.k, s.v, i32(pages), s.table, *wide)
    st.synchronize()
    # the last step's results from what the cache holds, and what it holds from the rows
    for slot in range(2):
        x = torch.cat(rows[slot])
        q, kx, vx = s.split(x, torch.arange(len(x)))
        mine = [i for i, p in enumerate(pages) if p[0] == slot]
        for w, y in zip(wide, (kx, vx)):
            got = w[mine].transpose(0, 1).reshape(s.G, -1, s.hd)[:, :len(x), :y.shape[2]].transpose(0, 1).double().cpu()
            # two roundings at most where the unit grew, of subnormal numbers alone: a step of the largest unit
            assert ((got - y).abs() <= y.abs() * 2.0 ** -4 + y.abs().amax() * 2.0 ** -17 + 1e-5).all()
        k, v = s.values(s.k, slot, len(x)), s.values(s.v, slot, len(x))
        want, moved = O.attend(q[-1:].cuda(), k, v, torch.ones(1, len(x), dtype=torch.bool), 0.1)
        compare(out[slot:slot + 1].view(1, s.H, s.vdim), want, moved, v.abs().max())


def test_captured_steps():
    """Two graphs of decode steps, replayed in turn on changing rows."""
    s = Setup(H=8, G=2, dim=64, slots=4, n_ctx=300, seed=29)
    t = Setup(H=8, G=2, dim=64, slots=4, n_ctx=300, seed=29)
    for c in (s, t):
        for slot in range(4):
            c.fill(slot, 60 + 50 * slot)
    xs, out = [torch.zeros(2, s.ld, device="cuda") for _ in range(2)], [torch.zeros(2, s.H * 64, device="cuda") for _ in range(2)]
    pos, slots = [i32([60, 110]), i32([160, 210])], [i32([0, 1]), i32([2, 3])]
    prep = s.prep()
    graphs = []
    cap = torch.cuda.Stream()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=cap):
            s.P.attn_decode8(xs[i], s.k, s.v, pos[i], slots[i], s.table, out[i], n_ctx=300, scale=0.2, pdl=True, **prep)
            pos[i] += 1
        graphs.append(g)
    at = [[60, 110], [160, 210]]
    for step in range(9):
        i = step % 2 if step < 6 else 1
        x = s.rnd(2, s.ld)
        xs[i].copy_(x)
        graphs[i].replay()
        want = torch.zeros_like(out[i])
        t.P.attn_decode8(x.cuda(), t.k, t.v, i32(at[i]), slots[i], t.table, want, n_ctx=300, scale=0.2, **prep)
        assert torch.equal(out[i], want)
        at[i] = [p + 1 for p in at[i]]
    used = s.table.reshape(-1).long()
    assert torch.equal(s.k.codes[used], t.k.codes[used]) and torch.equal(s.v.unit[used], t.v.unit[used])


def test_pages_far_into_a_large_cache():
    """Codes behind the first four billion."""
    G = 8
    first = (1 << 32) // (G * 64 * 128) + 7
    s = Setup(H=16, G=G, dim=128, slots=1, n_ctx=200, seed=31, first_page=first)
    s.fill(0, 150)
    x = s.rnd(1, s.ld)
    out = torch.zeros(1, s.H * 128, device="cuda")
    s.P.attn_decode8(x.cuda(), s.k, s.v, i32([150]), i32([0]), s.table, out, n_ctx=200, scale=0.1, **s.prep())
    at = s.table[0].long()
    k, v = ((torch.nan_to_num(c.numbers[at].float().double(), nan=0.0) * c.unit[at].double()[..., None, None]).transpose(0, 1).reshape(G, -1, 128)[:, :151] for c in (s.k, s.v))
    want, moved = O.attend(s.split(x, torch.tensor([150]))[0].cuda(), k, v, torch.ones(1, 151, dtype=torch.bool), 0.1)
    compare(out.view(1, s.H, 128), want, moved, v.abs().max())
    q, plan = torch.randn(3, s.H, 128, device="cuda"), s.P.portions8([(0, 3, 0, 148)], s.table)
    o = torch.zeros(3, s.H * 128, device="cuda", dtype=torch.bfloat16)
    s.P.attn_prompt8(q, s.k, s.v, plan, s.table, o, vdim=128, scale=0.1)
    want, moved = O.attend(q.double(), k, v, O.visible(torch.arange(148, 151), 151), 0.1)
    compare(o.view(3, s.H, 128), want, moved, v.abs().max())


@pytest.mark.parametrize("n", [5000, 33333])
def test_long_sequences(n):
    """One key near the start has nearly all of the weight; windows and chunks end elsewhere."""
    s = Setup(H=4, G=1, dim=64, norm="", n_rot=0, slots=1, n_ctx=n + 1, seed=n)
    s.fill(0, n)
    x = s.rnd(1, s.ld)
    target = s.values(s.k, 0, 71)[0, 70].float().cpu()
    x[0, :s.nq] = (target / target.norm() * 40).repeat(4)
    q = s.split(x, torch.tensor([n]))[0].cuda()
    for mask in (dict(), dict(window=300, keep=71), dict(chunk=1024), dict(window=4000, keep=5)):
        out = torch.zeros(1, 4 * 64, device="cuda")
        s.P.attn_decode8(x.cuda(), s.k, s.v, i32([n]), i32([0]), s.table, out, n_ctx=n + 1, scale=1.0, **s.prep(), **mask)
        k, v = s.values(s.k, 0, n + 1), s.values(s.v, 0, n + 1)
        want, moved = O.attend(q, k, v, O.visible(torch.tensor([n]), n + 1, **mask), 1.0)
        compare(out.view(1, 4, 64), want, moved, v.abs().max())


def test_refusals():
    s = Setup(H=4, G=2, dim=64)
    P, x = s.P, s.rnd(2, s.ld).cuda()
    q, pos, slots = torch.empty(2, 4, 64, device="cuda"), i32([0, 0]), i32([0, 1])
    prep = s.prep()
    before = s.k.codes.clone()

    def append(qkv=x, **kw):
        a = {**dict(k=s.k, v=s.v, table=s.table, q_out=q, positions=pos, slots=slots), **prep, **kw}
        P.append8(qkv, a.pop("k"), a.pop("v"), a.pop("table"), a.pop("q_out"), **a)

    other = P.Pages8.empty(4, 2, 128)
    for kw in (dict(qkv=x.half()), dict(qkv=x.cpu()), dict(qkv=x.t()), dict(v=other), dict(table=s.table.long()), dict(table=s.table[:, ::2]), dict(q_out=q[:1]), dict(q_out=q[..., :32]),
               dict(heads=3), dict(dim=65), dict(dim=0), dict(vdim=80), dict(v_off=400), dict(v_off=-1), dict(maps=2), dict(maps=3), dict(n_rot=66), dict(n_rot=3), dict(n_rot=-2),
               dict(freqs=s.f[:5]), dict(freqs=s.f.float()), dict(q_norm=None), dict(k_norm=s.held[1][:60]), dict(positions=None), dict(slots=slots[:1]), dict(slots=slots.long()),
               dict(append=False), dict(portions=P.portions8([(0, 2, 0, 0)], s.table)), dict(positions=None, slots=None, portions=P.portions8([(0, 3, 0, 0)], s.table))):
        with pytest.raises(ValueError):
            append(**kw)
    out = torch.zeros(2, 256, device="cuda", dtype=torch.bfloat16)
    plan = P.portions8([(0, 2, 0, 0)], s.table)
    for kw in (dict(out=out.half()), dict(out=out[:1]), dict(out=out[:, :250]), dict(out=out.t()), dict(vdim=65), dict(vdim=0), dict(chunk=3, window=4), dict(window=-1), dict(keep=-1), dict(chunk=-1),
               dict(softcap=-1.0), dict(q=q.bfloat16()), dict(q=q.cpu()), dict(q=q[:, :3]), dict(q=q[:1])):
        a = {**dict(q=q, k=s.k, v=s.v, portions=plan, table=s.table, out=out, vdim=64, scale=0.1), **kw}
        with pytest.raises(ValueError):
            P.attn_prompt8(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("portions"), a.pop("table"), a.pop("out"), **a)
    pages, wide = i32([[0, 0, 64, 0]]), [torch.zeros(1, 2, 64, 64, device="cuda", dtype=torch.float16) for _ in range(2)]
    for kw in (dict(pages=pages.cpu()), dict(pages=pages.long()), dict(pages=pages[:, :3]), dict(k_out=wide[0].bfloat16()), dict(v_out=wide[1][..., :32])):
        a = {**dict(k=s.k, v=s.v, pages=pages, table=s.table, k_out=wide[0], v_out=wide[1]), **kw}
        with pytest.raises(ValueError):
            P.read8(**a)
    assert torch.equal(before, s.k.codes) and (out == 0).all()
    append()
    append(x[:0], q_out=q[:0], positions=pos[:0], slots=slots[:0])          # no rows: nothing to do
    P.read8(s.k, s.v, pages[:0], s.table, wide[0][:0], wide[1][:0])
    P.attn_decode8(x[:0], s.k, s.v, pos[:0], slots[:0], s.table, out[:0], n_ctx=100, scale=0.1, **prep)


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("geometry", [GEOMETRIES[i] for i in (0, 1, 4, 8)])
def test_prompt_attention_with_32_bit_results(geometry, mask):
    """Many rows of several sequences, whose pages are not read out first."""
    from ollama_b200.ops import rows as R
    s = Setup(slots=3, n_ctx=1300, seed=37, **geometry)
    held = [0, 0, 0]
    for lens in ([260, 1, 64], [3, 600, 400]):
        parts, at = [], 0
        for slot in (1, 2, 0):
            parts.append((at, lens[slot], slot, held[slot]))
            at += lens[slot]
        x, q = s.rnd(at, s.ld), torch.empty(at, s.H, s.hd, device="cuda")
        plan = s.P.portions8(parts, s.table, **{n: mask[n] for n in mask if n != "softcap"})
        s.P.append8(x.cuda(), s.k, s.v, s.table, q, portions=plan, **s.prep())
        gate = ("element", "head")[at % 2]
        gv = s.rnd(at, s.H * s.vdim).cuda()
        out = torch.full((at, s.H * s.vdim + 8), 5.0, device="cuda")
        s.P.attn_prompt8(q, s.k, s.v, plan, s.table, out, vdim=s.vdim, scale=1.3 / math.sqrt(s.dim), gate=R.head_gate(gv, gate), **mask)
        assert (out[:, s.H * s.vdim:] == 5).all()
        for row, n, slot, p in parts:
            held[slot] += n
            pos = torch.arange(p, p + n)
            k, v = s.values(s.k, slot, p + n), s.values(s.v, slot, p + n)
            seen = O.visible(pos, p + n, **{m: mask[m] for m in mask if m != "softcap"})
            want, moved = O.attend(q[row:row + n, :, :s.dim].double(), k[..., :s.dim], v[..., :s.vdim], seen, 1.3 / math.sqrt(s.dim), mask.get("softcap", 0.0))
            f = torch.sigmoid(gv[row:row + n].double()).view(n, s.H, s.vdim) if gate == "element" else torch.sigmoid(gv[row:row + n, :s.H].double())[..., None]
            compare(out[row:row + n, :s.H * s.vdim].view(n, s.H, s.vdim), want * f, moved, v.abs().max())


@pytest.mark.parametrize("scale", [-0.2, 0.0, 0.2])
@pytest.mark.parametrize("softcap", [0.0, 3.0])
def test_scales_of_either_sign(scale, softcap):
    s = Setup(H=8, G=1, dim=64, norm="", n_rot=0, slots=1, n_ctx=700, seed=41)
    s.fill(0, 640, 2.0)
    k, v = s.values(s.k, 0, 640), s.values(s.v, 0, 640)
    for n, dtype in ((3, torch.bfloat16), (40, torch.float32), (300, torch.float32), (300, torch.bfloat16)):
        q = s.rnd(n, 8, 64).cuda()
        out = torch.zeros(n, 8 * 64, device="cuda", dtype=dtype)
        s.P.attn_prompt8(q, s.k, s.v, s.P.portions8([(0, n, 0, 640 - n)], s.table), s.table, out, vdim=64, scale=scale, softcap=softcap)
        want, moved = O.attend(q.double(), k, v, O.visible(torch.arange(640 - n, 640), 640), scale, softcap)
        compare(out.view(n, 8, 64), want, moved, v.abs().max())
    x = s.rnd(1, s.ld)
    out = torch.zeros(1, 8 * 64, device="cuda")
    s.P.attn_decode8(x.cuda(), s.k, s.v, i32([640]), i32([0]), s.table, out, n_ctx=700, scale=scale, softcap=softcap, **s.prep())
    k, v = s.values(s.k, 0, 641), s.values(s.v, 0, 641)
    want, moved = O.attend(s.split(x, torch.tensor([640]))[0].cuda(), k, v, torch.ones(1, 641, dtype=torch.bool), scale, softcap)
    compare(out.view(1, 8, 64), want, moved, v.abs().max())


def test_growing_scores():
    """Scores that rise from key to key by more than 2^8 a tile in their weights: what came before all but vanishes at each."""
    s = Setup(H=4, G=1, dim=64, norm="", n_rot=0, slots=1, n_ctx=1500, seed=43)
    x = s.rnd(1400, s.ld) * 0.1
    x[:, s.nq] = torch.arange(1400) / 16
    q = torch.empty(1400, 4, 64, device="cuda")
    s.P.append8(x.cuda(), s.k, s.v, s.table, q, portions=s.P.portions8([(0, 1400, 0, 0)], s.table), **s.prep())
    k, v = s.values(s.k, 0, 1400), s.values(s.v, 0, 1400)
    for n in (4, 200):
        for sign in (1.0, -1.0):
            y = s.rnd(n, 4, 64).cuda() * 0.1
            y[..., 0] = 2 * sign
            out = torch.zeros(n, 4 * 64, device="cuda")
            s.P.attn_prompt8(y, s.k, s.v, s.P.portions8([(0, n, 0, 1400 - n)], s.table), s.table, out, vdim=64, scale=1.0)
            want, moved = O.attend(y.double(), k, v, O.visible(torch.arange(1400 - n, 1400), 1400), 1.0)
            compare(out.view(n, 4, 64), want, moved, v.abs().max())


@pytest.mark.parametrize("n", [33, 40, 300])
def test_steps_of_many_rows(n):
    """More rows than a warp has lanes, and than a launch takes: each row's result is that of a call of its own."""
    s = Setup(H=4, G=2, dim=64, slots=n, n_ctx=128, seed=n)
    lens = [1 + (37 * i) % 120 for i in range(n)]
    t = Setup(H=4, G=2, dim=64, slots=n, n_ctx=128, seed=n)
    fill = s.rnd(sum(lens), s.ld).cuda()
    for c in (s, t):
        q, parts, at = torch.empty(len(fill), 4, 64, device="cuda"), [], 0
        for slot, m in enumerate(lens):
            parts.append((at, m, slot, 0))
            at += m
        for i in range(0, n, 100):
            some = parts[i:i + 100]
            a, b = some[0][0], some[-1][0] + some[-1][1]
            c.P.append8(fill[a:b], c.k, c.v, c.table, q[a:b], portions=c.P.portions8([(r - a, m, slot, 0) for r, m, slot, _ in some], c.table), **c.prep())
    x = s.rnd(n, s.ld).cuda()
    pos = [m if i % 9 else -1 for i, m in enumerate(lens)]
    out = torch.full((n, 256), 5.0, device="cuda")
    s.P.attn_decode8(x, s.k, s.v, i32(pos), i32(list(range(n))), s.table, out, n_ctx=128, scale=0.2, **s.prep())
    q = s.split(x.cpu(), torch.tensor(pos))[0]
    for i in range(n):
        if pos[i] < 0:
            assert (out[i] == 5).all()
            continue
        k, v = s.values(s.k, i, pos[i] + 1), s.values(s.v, i, pos[i] + 1)
        want, moved = O.attend(q[i:i + 1].cuda(), k, v, torch.ones(1, pos[i] + 1, dtype=torch.bool), 0.2)
        compare(out[i:i + 1].view(1, 4, 64), want, moved, v.abs().max())
    one = torch.zeros(1, 256, device="cuda")
    for i in range(1, n, 7):
        if pos[i] >= 0:
            t.P.attn_decode8(x[i:i + 1], t.k, t.v, i32(pos[i:i + 1]), i32([i]), t.table, one, n_ctx=128, scale=0.2, **t.prep())
            assert torch.allclose(one, out[i:i + 1], rtol=2.0 ** -9, atol=2.0 ** -9)
            at = t.table[i, :pos[i] // 64 + 1].long()
            assert torch.equal(s.k.codes[at], t.k.codes[at]) and torch.equal(s.v.unit[at], t.v.unit[at])


def test_values_that_are_no_number_in_many_rows():
    s = Setup(H=4, G=2, dim=64, norm="", n_rot=0, slots=1, n_ctx=600, seed=47)
    x = s.rnd(520, s.ld)
    x[450, s.v_off + 64 + 5] = math.nan               # KV head 1
    x[10, s.v_off + 3] = math.nan                     # KV head 0, seen through a kept key or not at all
    q = torch.empty(520, 4, 64, device="cuda")
    s.P.append8(x.cuda(), s.k, s.v, s.table, q, portions=s.P.portions8([(0, 520, 0, 0)], s.table), **s.prep())
    for mask in (dict(), dict(window=100), dict(window=100, keep=11), dict(window=100, keep=10), dict(chunk=64)):
        out = torch.zeros(500, 256, device="cuda")
        s.P.attn_prompt8(q[20:], s.k, s.v, s.P.portions8([(0, 500, 0, 20)], s.table, **mask), s.table, out, vdim=64, scale=0.1, **mask)
        seen = O.visible(torch.arange(20, 520), 520, **mask).cuda()
        o = out.view(500, 4, 64).isnan().any(-1)
        assert torch.equal(o[:, :2], seen[:, 10:11].expand(-1, 2)) and torch.equal(o[:, 2:], seen[:, 450:451].expand(-1, 2))


def test_read_back_without_what_is_no_number():
    from ollama_b200.ops import pages8 as P
    g = torch.Generator().manual_seed(5)
    codes = torch.randint(0, 256, (2, 2, 64, 64), generator=g, dtype=torch.int32).to(torch.uint8).cuda()
    codes[:, :, ::3] &= 0x77                            # some rows hold numbers alone
    c = P.Pages8(codes, torch.full((2, 2), 0.5, device="cuda"))
    out = [torch.empty(1, 2, 64, 64, device="cuda", dtype=torch.float16) for _ in range(2)]
    for clean in (0, 1):
        P.read8(c, c, i32([[0, 0, 64, 0]]), i32([[1]]), *out, clean=bool(clean))
        x = c.numbers[1].float() * 0.5
        none = x.isnan().any(-1, keepdim=True) & bool(clean)
        k, v = x.masked_fill(none, math.nan), x.masked_fill(none, 0.0)
        assert torch.equal(out[0][0].float().nan_to_num(nan=1e9), k.nan_to_num(nan=1e9)) and torch.equal(out[1][0].float().nan_to_num(nan=1e9), v.nan_to_num(nan=1e9))


@pytest.mark.parametrize("n", [6, 90, 400])
def test_captured_portions(n):
    """A portion's appending and attention in a graph, replayed over other rows, and beside a second graph of the same cache."""
    s, t = (Setup(H=8, G=2, dim=64, slots=2, n_ctx=1100, seed=53) for _ in range(2))
    for c in (s, t):
        for slot in range(2):
            c.fill(slot, 600)
    plans = [s.P.portions8([(0, n, slot, 600)], s.table) for slot in range(2)]
    xs, qs = torch.zeros(2, n, s.ld, device="cuda"), torch.zeros(2, n, 8, 64, device="cuda")
    outs, prep, cap, graphs = torch.zeros(2, n, 512, device="cuda", dtype=torch.bfloat16), s.prep(), torch.cuda.Stream(), []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=cap):
            s.P.append8(xs[i], s.k, s.v, s.table, qs[i], portions=plans[i], **prep)
            s.P.attn_prompt8(qs[i], s.k, s.v, plans[i], s.table, outs[i], vdim=64, scale=0.2)
        graphs.append(g)
    q, out = torch.empty(n, 8, 64, device="cuda"), torch.empty(n, 512, device="cuda", dtype=torch.bfloat16)
    for _ in range(2):
        x = torch.randn(2, n, s.ld, device="cuda")
        xs.copy_(x)
        for i in range(2):
            graphs[i].replay()
        for i in range(2):
            t.P.append8(x[i], t.k, t.v, t.table, q, portions=t.P.portions8([(0, n, i, 600)], t.table), **prep)
            t.P.attn_prompt8(q, t.k, t.v, t.P.portions8([(0, n, i, 600)], t.table), t.table, out, vdim=64, scale=0.2)
            assert torch.equal(outs[i], out)


def test_masks_of_any_size():
    """Windows, chunks and numbers of kept keys up to the largest integer are those that end with the sequence."""
    s = Setup(H=8, G=2, dim=64, slots=1, n_ctx=700, seed=59)
    s.fill(0, 640)
    most = 2 ** 31 - 1
    for n, dtype in ((1, torch.float32), (5, torch.float32), (300, torch.float32), (300, torch.bfloat16)):
        q, got = s.rnd(n, 8, 64).cuda(), []
        for mask in (dict(), dict(window=700), dict(window=most), dict(window=20, keep=700), dict(window=20, keep=most), dict(window=most, keep=most), dict(chunk=most)):
            out = torch.zeros(n, 512, device="cuda", dtype=dtype)
            s.P.attn_prompt8(q, s.k, s.v, s.P.portions8([(0, n, 0, 640 - n)], s.table, **mask), s.table, out, vdim=64, scale=0.1, **mask)
            got.append(out)
        assert all(torch.allclose(g.float(), got[0].float(), rtol=2.0 ** -7, atol=2.0 ** -9) for g in got)
    x = s.rnd(1, s.ld).cuda()
    got = []
    for mask in (dict(), dict(window=most), dict(window=20, keep=most), dict(chunk=most)):
        out = torch.zeros(1, 512, device="cuda")
        s.P.attn_decode8(x, s.k, s.v, i32([640]), i32([0]), s.table, out, n_ctx=700, scale=0.1, **s.prep(), **mask)
        got.append(out)
    assert all(torch.allclose(g, got[0], rtol=2.0 ** -9, atol=2.0 ** -9) for g in got)


def test_refusals_of_memory_that_does_not_fit():
    s = Setup(H=4, G=2, dim=64)
    P, plan, out, prep = s.P, s.P.portions8([(0, 2, 0, 0)], s.table), torch.zeros(2, 256, device="cuda"), s.prep()
    odd = lambda *shape, dtype=torch.float32: torch.zeros(math.prod(shape) + 1, device="cuda", dtype=dtype)[1:].view(shape)  # noqa: E731
    x = s.rnd(2, s.ld).cuda()
    with pytest.raises(ValueError):
        P.attn_prompt8(odd(2, 4, 64), s.k, s.v, plan, s.table, out, vdim=64, scale=0.1)
    for kw in (dict(softcap=math.inf), dict(softcap=math.nan), dict(out=torch.zeros(1, 256, device="cuda").expand(2, 256)), dict(out=torch.zeros(600, device="cuda").as_strided((2, 256), (200, 1)))):
        with pytest.raises(ValueError):
            P.attn_prompt8(**{**dict(q=torch.zeros(2, 4, 64, device="cuda"), k=s.k, v=s.v, portions=plan, table=s.table, out=out, vdim=64, scale=0.1), **kw})
    with pytest.raises(ValueError):
        P.append8(x, s.k, s.v, s.table, odd(2, 4, 64), portions=plan, **prep)
    with pytest.raises(ValueError):
        P.append8(x[:1].expand(2, s.ld), s.k, s.v, s.table, torch.zeros(2, 4, 64, device="cuda"), portions=plan, **prep)
    wide = [torch.zeros(1, 2, 64, 64, device="cuda", dtype=torch.float16) for _ in range(2)]
    with pytest.raises(ValueError):
        P.read8(s.k, s.v, odd(1, 4, dtype=torch.int32), s.table, *wide)
    with pytest.raises(ValueError):
        P.read8(s.k, s.v, i32([[0, 0, 64, 0]]), s.table, odd(1, 2, 64, 64, dtype=torch.float16), wide[1])
    assert (out == 0).all()
    # one row stands beside no other one: its step is not looked at
    one = torch.zeros(1, 256, device="cuda").as_strided((1, 256), (3, 1))
    P.attn_decode8(x[:1].as_strided((1, s.ld), (1, 1)), s.k, s.v, i32([0]), i32([0]), s.table, one, n_ctx=100, scale=0.1, **prep)
    assert (one != 0).any()
    # a plan that says less than its portions hold
    import dataclasses
    few, before = dataclasses.replace(s.P.portions8([(0, 40, 0, 0)], s.table), longest=1), torch.full((40, 256), 5.0, device="cuda")
    P.attn_prompt8(torch.zeros(40, 4, 64, device="cuda"), s.k, s.v, few, s.table, before, vdim=64, scale=0.1)
    assert (before == 5).all()


def test_refusal_of_too_many_rows():
    s, n = Setup(H=2, G=1, dim=64, slots=1, n_ctx=65600), 65536
    plan, out = s.P.portions8([(0, n, 0, 0)], s.table), torch.zeros(n, 128, device="cuda")
    with pytest.raises(ValueError, match="65536 rows"):
        s.P.attn_prompt8(torch.zeros(n, 2, 64, device="cuda"), s.k, s.v, plan, s.table, out, vdim=64, scale=0.1)
    with pytest.raises(ValueError, match="65536 rows"):
        s.P.attn_decode8(torch.zeros(n, s.ld, device="cuda"), s.k, s.v, torch.zeros(n, device="cuda", dtype=torch.int32), torch.zeros(n, device="cuda", dtype=torch.int32), s.table, out, n_ctx=100,
                         scale=0.1, **s.prep())
    assert (out == 0).all()
