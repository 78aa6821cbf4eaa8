"""Operators of the 8-bit paged cache, as cases for measuring: rows appended to it, its pages read back, decode attention and prompt
attention over it.

Keys and values of a sequence stand in pages of 64 positions, [page, KV head, position, column], as E4M3 numbers in units of a power of
two that each page has for each KV head.  Appending rows to a page sets its unit so that the largest magnitude in it fits; what the page
held is rounded to the new unit where that grew.  Cases are the sizes of the stack models' attention layers (heads x KV heads x columns:
4 x 2 x 64, 16 x 4 x 128, 32 x 8 x 128) and of the benchmark's batches and prompts; drawn ones have odd head sizes, masks and gates too.
"""
from __future__ import annotations

import math

import torch

own = False
PAGE = 64
LOW, HIGH = -15, 7               # exponents of a page's unit: with them every value of the cache is an f16 number too
TOP = 448.0                      # largest E4M3 magnitude
F8 = torch.float8_e4m3fn


def _case(name, op, heads, kv, dim, seqs, rows, ctx, **more) -> dict:
    """``seqs`` sequences with up to ``rows`` new rows each behind up to ``ctx`` cached positions."""
    return dict(name=name, op=op, heads=heads, kv=kv, dim=dim, vdim=dim, seqs=seqs, rows=rows, ctx=ctx, norm="row", window=0, keep=0, chunk=0, gate="", softcap=0.0) | more


def listed() -> list[dict]:
    return [
        # one user of a small test model: what a launch and the call cost
        _case("append 1", "append", 4, 2, 64, 1, 1, 201),
        # a decode step of sixteen sequences, each in the middle of a page of its own
        _case("append 16 slots", "append", 32, 8, 128, 16, 1, 1024, norm="head"),
        # one full chunk of a long prompt
        _case("append 2048 at 6144", "append", 32, 8, 128, 1, 2048, 6144),
        # a paragraph's cache, read back for a program that wants 16-bit rows
        _case("read 331", "read", 16, 4, 128, 1, 0, 331),
        # a server's eight long conversations
        _case("read 8 x 3001", "read", 32, 8, 128, 8, 0, 3001),
        # one user of a small test model
        _case("step, small", "decode", 4, 2, 64, 1, 1, 201),
        # one user's chat behind a long document
        _case("step, chat at 6144", "decode", 32, 8, 128, 1, 1, 6144),
        # a full server of a model with windows, kept first tokens and gated heads
        _case("step, 32 slots, window", "decode", 16, 4, 128, 32, 1, 1467, norm="head", window=1024, keep=8, gate="element"),
        # four users of whole books
        _case("step, 4 x 60000", "decode", 32, 8, 128, 4, 1, 60000),
        # drafted tokens that a target model scores
        _case("7 drafted at 901", "prompt", 32, 8, 128, 1, 7, 901),
        # a question of 64 tokens behind a book
        _case("64 rows at 30000", "prompt", 32, 8, 128, 1, 64, 30000),
        # one full chunk of a long prompt
        _case("chunk 2048 at 6144", "prompt", 32, 8, 128, 1, 2048, 6144),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    heads, kv, dim = rng.choice([(4, 2, 64), (16, 4, 128), (32, 8, 128), (6, 2, 48), (12, 4, 96), (8, 1, 100), (16, 16, 64)])
    op = rng.choice(["append", "read", "decode", "decode", "prompt", "prompt"])
    vdim = rng.choice([dim, dim, dim, dim - 8])
    mask = rng.choice(["", "", "window", "chunk"])
    more = dict(vdim=vdim, norm=rng.choice(["row", "head"]), gate=rng.choice(["", "", "element", "head"]), softcap=rng.choice([0.0, 0.0, 30.0]),
                window=_log(rng, 65, 2048) if mask == "window" else 0, keep=rng.randint(0, 80) if mask == "window" else 0, chunk=_log(rng, 100, 8192) if mask == "chunk" else 0)
    if op == "append":
        seqs = _log(rng, 1, 32)
        rows, ctx = rng.choice([1, _log(rng, 2, max(2, 2048 // seqs))]), rng.randint(0, 3000)
    elif op == "read":
        seqs = _log(rng, 1, 8)
        rows, ctx = 0, _log(rng, 17, 3001)
    elif op == "decode":
        seqs = _log(rng, 1, 32)
        rows, ctx = 1, _log(rng, 17, 100000 // seqs)
    else:
        seqs = rng.randint(1, 3)
        rows = _log(rng, 2, 1500 // seqs)
        ctx = rng.randint(0, 4000 if rows > 64 else 20000 // seqs)
    case = _case("", op, heads, kv, dim, seqs, rows, ctx, **more)
    del case["name"]
    return case


def _portions(case: dict) -> list[tuple[int, int, int, int]]:
    """(first row, rows, slot, position of the first row) of each sequence; the sequences are of uneven lengths."""
    out, at = [], 0
    for i in range(case["seqs"]):
        rows = case["rows"] - (i * 29) % max(1, case["rows"] // 2) if case["rows"] else 0
        out.append((at, rows, case["seqs"] - 1 - i, case["ctx"] - (i * 7919) % (case["ctx"] // 2 + 1)))
        at += rows
    return out


def _first(case: dict, pos: int) -> int:
    """First key that the query at a position sees, besides kept ones."""
    if case["chunk"]:
        return pos - pos % case["chunk"]
    return max(0, pos - case["window"] + 1) if case["window"] else 0


def work(case: dict) -> dict:
    H, G, d, v = case["heads"], case["kv"], case["dim"], case["vdim"]
    rows = keys = pairs = ends = 0
    for _, n, _, p in _portions(case):
        rows += n
        ends += p + n
        if n:
            lo = [_first(case, p + i) for i in range(n)]
            kept = [min(case["keep"], f) for f in lo]
            keys += p + n - lo[0] + kept[0]
            pairs += sum(p + i + 1 - f + k for i, (f, k) in enumerate(zip(lo, kept)))
    new = rows * (4 * (H * d + G * (d + v)) + G * (d + v))           # projections read, codes written
    if case["op"] == "append":
        return {"bytes": new + 4 * rows * H * d, "flops": 6 * rows * (H + G) * d}
    if case["op"] == "read":
        return {"bytes": 3 * ends * G * (d + v), "flops": 0}
    cache = keys * G * (d + v) + 8 * G * keys // PAGE
    rest = 2 * rows * H * v + 4 * rows * {"": 0, "element": H * v, "head": H}[case["gate"]]
    return {"bytes": cache + rest + (new if case["op"] == "decode" else 4 * rows * H * d), "flops": 2 * H * pairs * (d + v)}


# ---- inputs -----------------------------------------------------------------------------------------------------------------------
def _codes(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Pages [..., 64, columns] as codes and units."""
    top = x.abs().amax((-2, -1))
    m, e = torch.frexp(top / TOP)
    unit = torch.exp2(torch.where(m > 0.5, e, e - 1).clamp(LOW, HIGH).float())
    return (x / unit[..., None, None]).clamp(-TOP, TOP).to(F8).view(torch.uint8), unit


def prepare(case: dict, seed: int) -> dict:
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev).manual_seed(seed)
    H, G, d, v = case["heads"], case["kv"], case["dim"], case["vdim"]
    hd = 64 if max(d, v) <= 64 else 128
    parts = _portions(case)

    def rnd(*s):
        return torch.randn(*s, device=dev, generator=g)

    most = max(-(-(p + max(n, 1)) // PAGE) for _, n, _, p in parts)
    n_pages = case["seqs"] * most + 3
    order = torch.randperm(n_pages, device=dev, generator=g)[:case["seqs"] * most].to(torch.int32)
    s = dict(case=case, parts=parts, hd=hd, table=order.view(case["seqs"], most).contiguous())
    # keys have a few columns that stand out, as rotated ones do; pages differ in size
    column = 1.0 + 3.0 * (torch.rand(G, 1, d, device=dev, generator=g) > 0.94)
    for name, n in (("k", d), ("v", v)):
        s[name], s[name + "_unit"] = torch.empty(n_pages, G, PAGE, hd, device=dev, dtype=torch.uint8), torch.empty(n_pages, G, device=dev)
        for a in range(0, n_pages, 512):
            m = min(512, n_pages - a)
            x = torch.zeros(m, G, PAGE, hd, device=dev)
            x[..., :n] = rnd(m, G, PAGE, n) * torch.exp2(torch.rand(m, G, 1, 1, device=dev, generator=g) * 1.6 - 0.8)
            if name == "k":
                x[..., :n] *= column
            s[name][a:a + m], s[name + "_unit"][a:a + m] = _codes(x)
    total = sum(n for _, n, _, _ in parts)
    s["pos"] = torch.tensor([p + i for _, n, _, p in parts for i in range(n)], device=dev, dtype=torch.int32)
    s["slot"] = torch.tensor([t for _, n, t, _ in parts for _ in range(n)], device=dev, dtype=torch.int32)
    s["segs"] = torch.tensor(parts, device=dev, dtype=torch.int32)
    s["freqs"] = 500000.0 ** (-torch.arange(d // 2, device=dev, dtype=torch.float64) * 2 / d)
    s["scale"] = 1.5 / math.sqrt(d)
    ld = H * d + G * (d + v)
    s["g"] = rnd(total, H * v if case["gate"] == "element" else H) if case["gate"] else None
    if case["op"] in ("append", "decode"):
        s["qkv"] = rnd(total, ld)
        per = (H * d, G * d) if case["norm"] == "row" else (d, d)
        s["q_norm"], s["k_norm"] = 1.0 + 0.2 * rnd(per[0]), 1.0 + 0.2 * rnd(per[1])
    elif case["op"] == "prompt":
        s["q"] = torch.zeros(total, H, hd, device=dev)
        s["q"][..., :d] = rnd(total, H, d)
    # rows of the plain forms: sequence and row of each, sequences padded to the longest
    rows = max([n for _, n, _, _ in parts])
    s["seq"] = torch.tensor([i for i, (_, n, _, _) in enumerate(parts) for _ in range(n)], device=dev, dtype=torch.int64)
    s["row"] = torch.tensor([i for _, n, _, _ in parts for i in range(n)], device=dev, dtype=torch.int64)
    s["shape"] = (len(parts), rows)
    s["touched"] = torch.tensor(sorted({(t, b) for _, n, t, p in parts for b in range(p // PAGE, (p + n - 1) // PAGE + 1)}), device=dev, dtype=torch.int64).view(-1, 2)
    s["pages"] = torch.tensor([(t, b, min(PAGE, p + n - b * PAGE), 0) for _, n, t, p in parts for b in range(-(-(p + n) // PAGE))], device=dev, dtype=torch.int32)
    s["out"] = torch.zeros(total, H * v, device=dev, dtype=torch.bfloat16)
    s["q_out"] = torch.zeros(total, H, hd, device=dev)
    s["wide"] = [torch.zeros(len(s["pages"]), G, PAGE, hd, device=dev, dtype=torch.float16) for _ in range(2)] if case["op"] == "read" else None
    s["plan"] = None
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------------------
def _values(s: dict, name: str, at: torch.Tensor) -> torch.Tensor:
    return s[name][at].view(F8).float() * s[name + "_unit"][at][..., None, None]


def _rotated(x: torch.Tensor, pos: torch.Tensor, freqs: torch.Tensor) -> torch.Tensor:
    a = pos.double()[:, None] * freqs
    c, n, h = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None], len(freqs)
    lo, hi = x[..., :h], x[..., h:2 * h]
    return torch.cat([lo * c - hi * n, hi * c + lo * n, x[..., 2 * h:]], -1)


def _normed(s: dict, x: torch.Tensor, w: torch.Tensor, heads: int) -> torch.Tensor:
    if s["case"]["norm"] == "head":
        x = x.view(len(x), heads, -1)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
    return x.view(len(x), heads, -1)


def _append(s: dict) -> torch.Tensor:
    """Queries [rows, heads, columns] of the raw projections; keys and values go into the cache."""
    c = s["case"]
    H, G, d, v = c["heads"], c["kv"], c["dim"], c["vdim"]
    q, k, val = torch.split(s["qkv"], [H * d, G * d, G * v], 1)
    q = _rotated(_normed(s, q, s["q_norm"], H), s["pos"], s["freqs"])
    k = _rotated(_normed(s, k, s["k_norm"], G), s["pos"], s["freqs"])
    block, off = (s["pos"] // PAGE).long(), (s["pos"] % PAGE).long()
    page = s["table"][s["slot"].long(), block].long()
    touched = s["table"][s["touched"][:, 0], s["touched"][:, 1]].long()
    for name, x in (("k", k), ("v", val.reshape(len(val), G, v))):
        x = torch.nn.functional.pad(x, (0, s["hd"] - x.shape[2]))
        codes, unit = s[name], s[name + "_unit"]
        top = torch.zeros_like(unit).index_reduce_(0, page, x.abs().amax(2), "amax")[touched]
        fresh = torch.zeros(len(unit), device=unit.device).index_reduce_(0, page, (off == 0).float(), "amax")[touched] > 0
        m, e = torch.frexp(top / TOP)
        need = torch.exp2(torch.where(m > 0.5, e, e - 1).clamp(LOW, HIGH).float())
        old = unit[touched]
        new = torch.where(fresh[:, None], need, torch.maximum(old, need))
        held = codes[touched]
        codes[touched] = torch.where(new[..., None, None] > old[..., None, None], (held.view(F8).float() * (old / new)[..., None, None]).clamp(-TOP, TOP).to(F8).view(torch.uint8), held)
        unit[touched] = new
        codes[page, :, off] = (x / unit[page][..., None]).clamp(-TOP, TOP).to(F8).view(torch.uint8)
    return q


def _attend(s: dict, q: torch.Tensor) -> torch.Tensor:
    c = s["case"]
    H, G, d, v = c["heads"], c["kv"], c["dim"], c["vdim"]
    (S, R), slots = s["shape"], s["segs"][:, 2].long()
    k, val = (_values(s, n, s["table"][slots].long()).transpose(1, 2).flatten(2, 3) for n in "kv")           # [sequences, KV heads, keys, columns]
    rows = torch.zeros(S, R, H, d, device=q.device)
    rows[s["seq"], s["row"]] = q
    pos = (s["segs"][:, 3:4] + torch.arange(R, device=q.device))[..., None]
    x = rows.view(S, R, G, H // G, d).permute(0, 2, 3, 1, 4).reshape(S, G, H // G * R, d) @ k[..., :d].transpose(2, 3) * s["scale"]
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    at = torch.arange(k.shape[2], device=q.device)
    low = pos - pos % c["chunk"] if c["chunk"] else (pos - c["window"] + 1).clamp(min=0) if c["window"] else torch.zeros_like(pos)
    seen = (at <= pos) & ((at >= low) | (at < (c["keep"] if c["window"] else 0)))
    x = x.view(S, G, H // G, R, -1).masked_fill_(~seen[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = (x / x.sum(-1, keepdim=True)).flatten(2, 3)
    # a masked key counts nothing, whatever its page holds
    o = (x @ torch.nan_to_num(val[..., :v])).view(S, G, H // G, R, v).permute(0, 3, 1, 2, 4).reshape(S, R, H, v)[s["seq"], s["row"]]
    if c["gate"]:
        o = o * torch.sigmoid(s["g"].view(len(o), H, -1))
    return o.reshape(len(o), H * v).to(torch.bfloat16)


def _cache(s: dict) -> dict:
    """The cache as it is: E4M3 numbers and the units they count in."""
    return {"k": s["k"].view(F8), "v": s["v"].view(F8), "k_unit": s["k_unit"], "v_unit": s["v_unit"]}


def _plain(s: dict):
    c = s["case"]
    if c["op"] == "append":
        q = _append(s)
        return {"q": torch.nn.functional.pad(q, (0, s["hd"] - c["dim"])), **_cache(s)}
    if c["op"] == "read":
        at = s["table"][s["pages"][:, 0].long(), s["pages"][:, 1].long()].long()
        inside = (torch.arange(PAGE, device=at.device) < s["pages"][:, 2:3])[:, None, :, None]
        return [torch.where(inside, _values(s, n, at), 0.0).to(torch.float16) for n in "kv"]
    if c["op"] == "decode":
        return {"out": _attend(s, _append(s)), **_cache(s)}
    return _attend(s, s["q"][..., :c["dim"]])


# ---- the framework's calls --------------------------------------------------------------------------------------------------------
def _own(s: dict):
    from ollama_b200.ops import pages8 as P
    from ollama_b200.ops import rows as O
    c = s["case"]
    H, G, d, v = c["heads"], c["kv"], c["dim"], c["vdim"]
    if s["plan"] is None:            # what an engine keeps over its steps: the pages of a layer, and for a prompt the portions of the step
        s["plan"] = {"k": P.Pages8(s["k"], s["k_unit"]), "v": P.Pages8(s["v"], s["v_unit"]),
                     "gate": O.head_gate(s["g"], c["gate"]) if c["gate"] else O.NO_GATE,
                     "portions": P.portions8(s["parts"], s["table"], window=c["window"], keep=c["keep"], chunk=c["chunk"]) if c["op"] in ("append", "prompt") else None}
    p = s["plan"]
    k, val = p["k"], p["v"]
    mask = dict(scale=s["scale"], softcap=c["softcap"], chunk=c["chunk"], window=c["window"], keep=c["keep"], gate=p["gate"])
    if c["op"] == "read":
        P.read8(k, val, s["pages"], s["table"], *s["wide"])
        return s["wide"]
    if c["op"] == "prompt":
        P.attn_prompt8(s["q"], k, val, p["portions"], s["table"], s["out"], vdim=v, **mask)
        return s["out"]
    prep = dict(heads=H, dim=d, vdim=v, q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6, freqs=s["freqs"], n_rot=2 * len(s["freqs"]), head_norm=c["norm"] == "head")
    if c["op"] == "append":
        if c["rows"] == 1:
            P.append8(s["qkv"], k, val, s["table"], s["q_out"], positions=s["pos"], slots=s["slot"], **prep)
        else:
            P.append8(s["qkv"], k, val, s["table"], s["q_out"], portions=p["portions"], **prep)
        return {"q": s["q_out"], **_cache(s)}
    P.attn_decode8(s["qkv"], k, val, s["pos"], s["slot"], s["table"], s["out"], n_ctx=c["ctx"] + 1, **prep, **mask)
    return {"out": s["out"], **_cache(s)}


def run(state: dict):
    return _own(state) if own else _plain(state)


# ---- the definition, in 64 bits ---------------------------------------------------------------------------------------------------
def _e4m3(x: torch.Tensor) -> torch.Tensor:
    """The nearest E4M3 numbers, ties to even: four bits from 2^-6 on, steps of 2^-9 below."""
    a = x.abs().clamp(max=TOP)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.sign(x) * torch.round(a / step) * step


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    H, G, d, v, hd = case["heads"], case["kv"], case["dim"], case["vdim"], s["hd"]
    table, dev = s["table"].tolist(), s["k"].device
    held = {n: s[n].view(F8).double() for n in "kv"}
    unit = {n: s[n + "_unit"].double() for n in "kv"}
    if case["op"] == "read":
        out = {n: torch.zeros(len(s["pages"]), G, PAGE, hd, device=dev, dtype=torch.float64) for n in "kv"}
        for i, (t, b, n, _) in enumerate(s["pages"].tolist()):
            for name in "kv":
                out[name][i, :, :n] = held[name][table[t][b], :, :n] * unit[name][table[t][b]][:, None, None]
        return [out["k"], out["v"]]
    if case["op"] == "prompt":
        q = s["q"][..., :d].double()
    else:
        x = s["qkv"].double()
        q, k, val = x[:, :H * d].view(-1, H, d), x[:, H * d:(H + G) * d].view(-1, G, d), x[:, (H + G) * d:].view(-1, G, v)
        over = -1 if case["norm"] == "head" else (-2, -1)

        def turned(y, w):
            w = w.double().view(1, -1, d)
            y = y / ((y ** 2).mean(over, keepdim=True) + 1e-6).sqrt() * w
            z = torch.polar(torch.ones((), dtype=torch.float64, device=dev), s["pos"].double()[:, None, None] * s["freqs"])
            h = d // 2
            z = torch.complex(y[..., :h], y[..., h:2 * h].contiguous()) * z
            return torch.cat([z.real, z.imag, y[..., 2 * h:]], -1)

        q, k = turned(q, s["q_norm"]), turned(k, s["k_norm"])
        for row, n, t, p in s["parts"]:
            for b in range(p // PAGE, (p + n - 1) // PAGE + 1):
                lo, hi = max(p, b * PAGE), min(p + n, (b + 1) * PAGE)
                page = table[t][b]
                for name, y in (("k", k), ("v", val)):
                    y = y[row + lo - p:row + hi - p].transpose(0, 1)
                    need = torch.full((G,), 2.0 ** HIGH, device=dev, dtype=torch.float64)
                    for e in range(HIGH, LOW - 1, -1):
                        need = torch.where(y.abs().amax((1, 2)) <= TOP * 2.0 ** e, 2.0 ** e, need)
                    new = need if lo % PAGE == 0 else torch.maximum(need, unit[name][page])
                    if lo % PAGE or hi - lo < PAGE:
                        grown = new > unit[name][page]
                        held[name][page] = torch.where(grown[:, None, None], _e4m3(held[name][page] * (unit[name][page] / new)[:, None, None]), held[name][page])
                    unit[name][page] = new
                    held[name][page, :, lo - b * PAGE:hi - b * PAGE] = 0
                    held[name][page, :, lo - b * PAGE:hi - b * PAGE, :y.shape[2]] = _e4m3(y / new[:, None, None])
    cache = {"k": held["k"], "v": held["v"], "k_unit": unit["k"], "v_unit": unit["v"]}
    if case["op"] == "append":
        full = torch.zeros(len(q), H, hd, device=dev, dtype=torch.float64)
        full[..., :d] = q
        return {"q": full, **cache}
    out = torch.zeros(len(q), H, v, device=dev, dtype=torch.float64)
    for row, n, t, p in s["parts"]:
        at = torch.tensor(table[t], device=dev)
        keys, vals = ((held[m][at] * unit[m][at][..., None, None]).transpose(0, 1).reshape(G, -1, hd)[:, :p + n] for m in "kv")
        for a in range(0, n, 512):
            z = min(n, a + 512)
            seen = torch.zeros(z - a, p + n, device=dev, dtype=torch.bool)
            for i in range(a, z):
                seen[i - a, _first(case, p + i):p + i + 1] = True
                seen[i - a, :min(case["keep"] if case["window"] else 0, p + i + 1)] = True
            for h in range(H):
                x = q[row + a:row + z, h] @ keys[h * G // H, :, :d].T * s["scale"]
                if case["softcap"]:
                    x = case["softcap"] * torch.tanh(x / case["softcap"])
                out[row + a:row + z, h] = torch.softmax(torch.where(seen, x, -math.inf), 1) @ vals[h * G // H, :, :v]
    if case["gate"]:
        out *= torch.sigmoid(s["g"].double()).view(len(out), H, -1)
    out = out.view(len(out), H * v)
    return {"out": out, **cache} if case["op"] == "decode" else out
