"""Operators of a 4-bit K/V cache and of packed prompts, as cases for measuring: rows appended to the cache and read back, single tokens' attention over it, attention of
prompts of different lengths in one call, over the cache or over 16-bit keys and values.

A cached row holds 32 columns at a time as integers 0 .. 15 under one f16 scale d: a value is d (code - 8), and d is minus an eighth of the value of largest magnitude (of
two, the negative one).  Cases have the heads (heads x KV heads x columns) of this repository's models and tests, its benchmark's batches and prompts, and other lengths of
context; drawn ones have uneven groups, windows, soft caps and attention sinks too.
"""
from __future__ import annotations

import math

import torch

own = False
BLOCK = 32                       # columns under one scale
TOP = 8188.0                     # largest scale: eight times it is an f16 number


def _case(name, op, heads, kv, dim, seqs, rows, ctx, **more) -> dict:
    """``seqs`` sequences with up to ``rows`` new rows each behind up to ``ctx`` cached positions."""
    return dict(name=name, op=op, heads=heads, kv=kv, dim=dim, seqs=seqs, rows=rows, ctx=ctx, window=0, softcap=0.0, sinks=False, norm=False, neox=True, rot=dim, kind="f16") | more


def listed() -> list[dict]:
    return [
        # one user of a small test model: what a launch and the call cost
        _case("append 1", "append", 4, 2, 64, 1, 1, 201),
        # a step of sixteen sequences of a model with normalised heads
        _case("append 16 slots", "append", 32, 8, 128, 16, 1, 1024, norm=True),
        # one full chunk of a long prompt
        _case("append 2048 at 6144", "append", 32, 8, 128, 1, 2048, 6144, neox=False),
        # one user of a small test model, from the raw projections on
        _case("step, small", "step", 4, 2, 64, 1, 1, 201),
        # one user's chat behind a long document
        _case("step, chat at 6144", "step", 32, 8, 128, 1, 1, 6144, neox=False),
        # a full server of a model with windows and attention sinks
        _case("32 slots, window", "decode", 64, 8, 64, 32, 1, 1467, window=1024, sinks=True),
        # four users of whole books
        _case("4 x 60000", "decode", 32, 8, 128, 4, 1, 60000),
        # drafted tokens that a target model scores
        _case("7 drafted at 901", "prompt", 32, 8, 128, 1, 7, 901),
        # a question of 64 tokens behind a book
        _case("64 rows at 30000", "prompt", 32, 8, 128, 1, 64, 30000),
        # one full chunk of a long prompt
        _case("chunk 2048 at 6144", "prompt", 32, 8, 128, 1, 2048, 6144),
        # a server's short requests that came together, without a cache
        _case("9 short prompts", "packed", 32, 8, 128, 9, 331, 0, kind="bf16"),
        # long prompts that came together
        _case("5 prompts of 4096", "packed", 32, 8, 128, 5, 4096, 0),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    heads, kv, dim = rng.choice([(4, 2, 64), (16, 4, 128), (32, 8, 128), (64, 8, 64), (14, 2, 64), (28, 4, 128), (8, 1, 128), (16, 16, 64), (40, 2, 128)])
    op = rng.choice(["append", "step", "decode", "prompt", "prompt", "packed"])
    more = dict(window=_log(rng, 20, 3000) if rng.random() < 0.4 else 0, softcap=rng.choice([0.0, 0.0, 30.0]), sinks=rng.random() < 0.3, norm=rng.random() < 0.5,
                neox=rng.random() < 0.5, rot=rng.choice([dim, dim, dim // 2]), kind=rng.choice(["f16", "bf16"]))
    if op == "append":
        seqs = _log(rng, 1, 32)
        rows, ctx = rng.choice([1, _log(rng, 2, max(2, 2048 // seqs))]), rng.randint(0, 3000)
    elif op in ("step", "decode"):
        seqs = _log(rng, 1, 32)
        rows, ctx = 1, _log(rng, 1, 100000 // seqs)
    elif op == "prompt":
        seqs = rng.randint(1, 4)
        rows = _log(rng, 2, 1500 // seqs)
        ctx = rng.randint(0, 4000 if rows > 64 else 20000 // seqs)
    else:
        seqs = _log(rng, 1, 16)
        rows, ctx = _log(rng, 1, 4096 // seqs), 0
    case = _case("", op, heads, kv, dim, seqs, rows, ctx, **more)
    del case["name"]
    return case


def _portions(case: dict) -> list[tuple[int, int, int, int, int]]:
    """(first row, rows, slot, position of the first row, cache row of position 0) of each sequence; the sequences are of uneven lengths."""
    out, at = [], 0
    for i in range(case["seqs"]):
        rows = case["rows"] - (i * 29 * (case["rows"] // 97 + 1)) % max(1, 3 * case["rows"] // 4)
        if case["op"] == "packed":
            out.append((at, rows, 0, 0, at))
        else:
            out.append((at, rows, case["seqs"] - i, case["ctx"] - (i * 7919) % (case["ctx"] // 2 + 1), 0))
        at += rows
    return out


def _first(case: dict, pos: int) -> int:
    """First key that the query at a position sees."""
    return max(0, pos - case["window"] + 1) if case["window"] else 0


def _pairs(case: dict) -> tuple[int, int]:
    """Keys that some query of their sequence sees, and pairs of a query row and a key that it sees."""
    keys = pairs = 0
    for _, n, _, p, _ in _portions(case):
        keys += p + n - _first(case, p)
        pairs += sum(p + i + 1 - _first(case, p + i) for i in range(n))
    return keys, pairs


def work(case: dict) -> dict:
    H, G, d = case["heads"], case["kv"], case["dim"]
    rows = sum(n for _, n, _, _, _ in _portions(case))
    held = 2 * G * (d // 2 + d // 16)             # bytes of a cached token
    if case["op"] == "append":                    # projections in; queries, cached rows and their values out
        return {"bytes": rows * (4 * (H + 2 * G) * d + 2 * H * d + 2 * held + 4 * G * d), "flops": 0}
    keys, pairs = _pairs(case)
    if case["op"] == "step":
        return {"bytes": rows * (4 * (H + 2 * G) * d + 2 * H * d + held + 4 * G * d) + keys * held, "flops": 4 * H * d * pairs}
    return {"bytes": rows * 4 * H * d + keys * (4 * G * d if case["op"] == "packed" else held), "flops": 4 * H * d * pairs}


# ---- inputs -----------------------------------------------------------------------------------------------------------------------
def _encode(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Integers 0 .. 15 [..., blocks, 32] and f16 scales [..., blocks]."""
    x = x.view(*x.shape[:-1], -1, BLOCK)
    hi, lo = x.amax(-1), x.amin(-1)
    d = (-torch.where(hi > -lo, hi, lo) / 8).clamp(-TOP, TOP).to(torch.float16)
    w = d.float()[..., None]
    return torch.where(w != 0, torch.round(x / w) + 8, 8.0).clamp(0, 15).to(torch.uint8), d


def _pack(codes: torch.Tensor) -> torch.Tensor:
    """A row's codes as its bytes [..., columns / 2].  Eight neighbouring columns are a 32-bit word, column 2 i of them in bits 4 i .., column 2 i + 1 in bits 16 + 4 i ..;
    word j of every block comes before word j + 1 of any."""
    c = codes.unflatten(-1, (4, 4, 2)).transpose(-4, -3).to(torch.uint8)                    # [..., word, block, pair, of it]
    c = c.transpose(-1, -2)                                                                 # even columns, then odd ones
    return (c[..., 0::2] | c[..., 1::2] << 4).flatten(-4)


def _unpack(rows: torch.Tensor) -> torch.Tensor:
    """The other way, [..., blocks, 32]."""
    c = rows.unflatten(-1, (4, -1, 2, 2))                                                   # [..., word, block, even or odd, byte]
    c = torch.stack([c & 15, c >> 4], -1).flatten(-2)                                       # [..., word, block, even or odd, pair]
    return c.transpose(-1, -2).transpose(-4, -3).flatten(-3)


def prepare(case: dict, seed: int) -> dict:
    dev = "cuda"
    g = torch.Generator(dev).manual_seed(seed)

    def rnd(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    H, G, d, parts = case["heads"], case["kv"], case["dim"], _portions(case)
    total = sum(n for _, n, _, _, _ in parts)
    s = dict(case=case, parts=parts, plan=None, scale=1.5 / math.sqrt(d), sinks=rnd(H) * 2 if case["sinks"] else None)
    # keys have a few columns that stand out, as rotated ones do; rows differ in size
    column = 1.0 + 3.0 * (torch.rand(1, 1, d, device=dev, generator=g) > 0.94)
    if case["op"] == "packed":
        t = torch.float16 if case["kind"] == "f16" else torch.bfloat16
        s["q"], s["k"], s["v"] = rnd(total, H, d).to(t), (rnd(total, G, d) * column).to(t), rnd(total, G, d).to(t)
    else:
        slots, n_ctx = case["seqs"] + 1, max(p + n for _, n, _, p, _ in parts) + 5
        for name in "kv":
            s[name] = torch.empty(slots, G, n_ctx, d // 2, device=dev, dtype=torch.uint8)
            s[name + "_scale"] = torch.empty(slots, G, n_ctx, d // BLOCK, device=dev, dtype=torch.float16)
            for i in range(slots):
                x = rnd(G, n_ctx, d) * torch.exp2(torch.rand(G, n_ctx, 1, device=dev, generator=g) * 1.6 - 0.8)
                codes, s[name + "_scale"][i] = _encode(x * column if name == "k" else x)
                s[name][i] = _pack(codes)
        s["freqs"] = (500000.0 ** (-torch.arange(case["rot"] // 2, device=dev, dtype=torch.float64) * 2 / case["rot"])).float()
        s["norms"] = [1.0 + 0.2 * rnd(d) for _ in range(2)] if case["norm"] else None
        if case["op"] in ("append", "step"):
            s["qkv"] = rnd(total, (H + 2 * G) * d)
        else:
            s["q"] = rnd(total, H, d).to(torch.float16 if case["kind"] == "f16" else torch.float32)
    s["pos"] = torch.tensor([p + i for _, n, _, p, _ in parts for i in range(n)], device=dev, dtype=torch.int32)
    s["slot"] = torch.tensor([t for _, n, t, _, _ in parts for _ in range(n)], device=dev, dtype=torch.int32)
    # rows of the plain forms: sequence and row of each, sequences padded to the longest
    s["seq"] = torch.tensor([i for i, p in enumerate(parts) for _ in range(p[1])], device=dev)
    s["row"] = torch.tensor([i for p in parts for i in range(p[1])], device=dev)
    s["segs"] = torch.tensor(parts, device=dev)
    s["shape"] = (len(parts), max(p[1] for p in parts), max(p[1] + p[3] for p in parts))
    s["out"] = torch.zeros(total, H * d, device=dev, dtype=torch.bfloat16)
    s["q_out"] = torch.zeros(total, H, d, device=dev, dtype=torch.float16)
    s["rows"] = [torch.zeros(total, G, d, device=dev, dtype=torch.float16) for _ in range(2)]
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------------------
def _values(s: dict, name: str, *at) -> torch.Tensor:
    """Cached rows [..., columns] as they are held."""
    return ((_unpack(s[name][at]).float() - 8) * s[name + "_scale"][at].float()[..., None]).flatten(-2)


def _append(s: dict) -> torch.Tensor:
    """Queries [rows, heads, columns] of the raw projections; keys and values go into the cache."""
    c = s["case"]
    H, G, d = c["heads"], c["kv"], c["dim"]
    q, k, v = s["qkv"].view(-1, H + 2 * G, d).split([H, G, G], 1)
    a = s["pos"].double()[:, None, None] * s["freqs"].double()
    cos, sin = torch.cos(a).float(), torch.sin(a).float()

    def turned(x, w):
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        x, rest = x.split([c["rot"], d - c["rot"]], -1)
        x0, x1 = x.chunk(2, -1) if c["neox"] else (x[..., 0::2], x[..., 1::2])
        x = [x0 * cos - x1 * sin, x0 * sin + x1 * cos]
        return torch.cat([torch.cat(x, -1) if c["neox"] else torch.stack(x, -1).flatten(-2), rest], -1)

    w = s["norms"] or (None, None)
    for name, x in (("k", turned(k, w[1])), ("v", v)):
        codes, scale = _encode(x)
        s[name][s["slot"], :, s["pos"]] = _pack(codes)
        s[name + "_scale"][s["slot"], :, s["pos"]] = scale
    return turned(q, w[0])


def _attend(s: dict, q: torch.Tensor) -> torch.Tensor:
    c = s["case"]
    H, G, d = c["heads"], c["kv"], c["dim"]
    S, R, N = s["shape"]
    if c["op"] == "packed":
        at = (s["segs"][:, 4:5] + torch.arange(N, device=q.device)).clamp(max=len(q) - 1)
        k, v = (s[n][at].float().transpose(1, 2) for n in "kv")                              # [sequences, KV heads, keys, columns]
    else:
        k, v = (_values(s, n, s["segs"][:, 2], slice(None), slice(0, N)) for n in "kv")
    rows = torch.zeros(S, R, H, d, device=q.device)
    rows[s["seq"], s["row"]] = q.float()
    pos = (s["segs"][:, 3:4] + torch.arange(R, device=q.device))[..., None]
    x = rows.view(S, R, G, H // G, d).permute(0, 2, 3, 1, 4).reshape(S, G, H // G * R, d) @ k.transpose(2, 3) * s["scale"]
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    at = torch.arange(N, device=q.device)
    seen = (at <= pos) & (at >= (pos - c["window"] + 1 if c["window"] else torch.zeros_like(pos)))
    x = x.view(S, G, H // G, R, N).masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(G, H // G, 1, 1)
        top = torch.maximum(top, sink)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top)
    x = (x / total).flatten(2, 3)
    o = (x @ v).view(S, G, H // G, R, d).permute(0, 3, 1, 2, 4).reshape(S, R, H, d)[s["seq"], s["row"]]
    return o.reshape(len(o), H * d).to(torch.bfloat16)


def _appended(s: dict) -> dict:
    """The new rows as the cache holds them."""
    return {n: _values(s, n, s["slot"], slice(None), s["pos"]).to(torch.float16) for n in "kv"}


def _plain(s: dict):
    op = s["case"]["op"]
    if op == "append":
        return {"q": _append(s).to(torch.float16), **_appended(s)}
    if op == "step":
        return {"out": _attend(s, _append(s)), **_appended(s)}
    return _attend(s, s["q"])


# ---- the framework's calls --------------------------------------------------------------------------------------------------------
def _own(s: dict):
    from ollama_b200.ops import kv4
    c = s["case"]
    if s["plan"] is None:            # what an engine keeps over its steps: a layer's cache, and the portions of a step for all its layers
        cached = c["op"] != "packed"
        s["plan"] = {n: kv4.Cache4(s[n], s[n + "_scale"]) if cached else s[n].transpose(0, 1)[None] for n in "kv"}
        if c["op"] in ("prompt", "packed"):
            s["plan"]["portions"] = kv4.portions4(s["parts"], c["heads"], s["plan"]["k"], window=c["window"])
    p = s["plan"]
    k, v = p["k"], p["v"]
    mask = dict(scale=s["scale"], softcap=c["softcap"], window=c["window"], sinks=s["sinks"])
    if c["op"] == "prompt":
        kv4.attn_prompt4(s["q"], k, v, p["portions"], s["out"], **mask)
        return s["out"]
    if c["op"] == "packed":
        kv4.attn_packed(s["q"], k, v, p["portions"], s["out"], **mask)
        return s["out"]
    if c["op"] == "decode":
        kv4.attn_decode4(s["q"], k, v, s["pos"], s["slot"], s["out"], **mask)
        return s["out"]
    w = s["norms"] or (None, None)
    prep = dict(heads=c["heads"], inv_freq=s["freqs"], n_rot=c["rot"], neox=c["neox"], q_norm=w[0], k_norm=w[1], eps=1e-6)
    if c["op"] == "append":
        kv4.append4(s["qkv"], k, v, s["pos"], s["slot"], s["q_out"], **prep)
        kv4.read4(k, v, s["pos"], s["slot"], *s["rows"])
        return {"q": s["q_out"], "k": s["rows"][0], "v": s["rows"][1]}
    kv4.attn_step4(s["qkv"], k, v, s["pos"], s["slot"], s["out"], **prep, **mask)
    kv4.read4(k, v, s["pos"], s["slot"], *s["rows"])
    return {"out": s["out"], "k": s["rows"][0], "v": s["rows"][1]}


def run(state: dict):
    return _own(state) if own else _plain(state)


# ---- the definition, in 64 bits ---------------------------------------------------------------------------------------------------
def _held(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """Values of cached rows, column by column from their bits."""
    rows, d = codes.long(), 2 * codes.shape[-1]
    out = torch.empty(*rows.shape[:-1], d, device=rows.device, dtype=torch.float64)
    for col in range(d):
        block, word, pair, odd = col // 32, col % 32 // 8, col % 8 // 2, col % 2
        at = 4 * (word * (d // 32) + block) + 2 * odd + pair // 2
        out[..., col] = ((rows[..., at] >> 4 * (pair % 2) & 15) - 8) * scale[..., block].double()
    return out


def _rounded(x: torch.Tensor) -> torch.Tensor:
    """Rows [rows, heads, columns] as a cache holds them."""
    y = x.reshape(len(x), x.shape[1], -1, 32)
    far = torch.gather(y, -1, y.abs().argmax(-1, keepdim=True))
    d = (-far / 8).to(torch.float16).double()
    return torch.where(d == 0, 0.0, d * (torch.round(y / d).clamp(-8, 7))).reshape(x.shape)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    H, G, d, parts = case["heads"], case["kv"], case["dim"], s["parts"]
    if 4 * H * d * _pairs(case)[1] > 2e12:
        return None
    new = {}
    if case["op"] in ("append", "step"):
        x = s["qkv"].double().view(-1, H + 2 * G, d)
        q, k, v = x[:, :H], x[:, H:H + G], x[:, H + G:]
        h = case["rot"] // 2
        z = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), s["pos"].double()[:, None, None] * s["freqs"].double())
        first = torch.arange(h, device=x.device) * (1 if case["neox"] else 2)
        second = first + (h if case["neox"] else 1)

        def turned(y, w):
            if w is not None:
                y = y / ((y ** 2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
            t = torch.complex(y[..., first], y[..., second]) * z
            y = y.clone()
            y[..., first], y[..., second] = t.real, t.imag
            return y

        w = s["norms"] or (None, None)
        q = turned(q, w[0])
        new = {"k": _rounded(turned(k, w[1])), "v": _rounded(v)}
        if case["op"] == "append":
            return {"q": q, **new}
    else:
        q = s["q"].double()
    out = torch.zeros(len(q), H, d, device=q.device, dtype=torch.float64)
    for row, n, t, p, base in parts:
        if case["op"] == "packed":
            keys, vals = (s[m][base:base + p + n].double().transpose(0, 1) for m in "kv")
        else:
            keys, vals = (_held(s[m][t, :, :p + n], s[m + "_scale"][t, :, :p + n]) for m in "kv")
        if new:
            keys[:, p:], vals[:, p:] = new["k"][row:row + n].transpose(0, 1), new["v"][row:row + n].transpose(0, 1)
        for a in range(0, n, 1024):
            z = min(n, a + 1024)
            at, pos = torch.arange(p + n, device=q.device), torch.arange(p + a, p + z, device=q.device)[:, None]
            seen = (at <= pos) & (at > pos - case["window"]) if case["window"] else at <= pos
            for h in range(H):
                x = q[row + a:row + z, h] @ keys[h * G // H].T * s["scale"]
                if case["softcap"]:
                    x = case["softcap"] * torch.tanh(x / case["softcap"])
                x = x.masked_fill(~seen, -math.inf)
                if s["sinks"] is not None:
                    x = torch.cat([x, s["sinks"][h].double().expand(z - a, 1)], 1)
                out[row + a:row + z, h] = torch.softmax(x, 1)[:, :p + n] @ vals[h * G // H]
    out = out.view(len(out), H * d)
    return {"out": out, **new} if case["op"] == "step" else out
