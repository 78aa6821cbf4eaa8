"""Models under OLLAMA_KV_CACHE_TYPE=int4: every layer's attention head by head against 64 bits, windows in the native pass, launches, served tokens, what a bench line says of the cache."""
import dataclasses

import pytest
import torch

import kv4_oracle as O
from test_int4_engine_gpu import Near, build, four_bits, status  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def tokens(n, seed):
    return torch.randint(259, 4096, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def assert_layer(eng, i, qkv, pos, slots, out, wide):
    """A layer's new cache rows and its results [rows, H * hd] from the raw projections, by the model's own settings."""
    c, L = eng.cfg, eng.layers[i]
    H, G, d = c.n_heads, c.n_kv_heads, c.head_dim
    local = c.layer_is_swa(i) and c.rope_base_local > 0
    inv, mscale = (eng.inv_freq_local, 1.0) if local else (eng.inv_freq, eng.mscale)
    q, k, v = qkv.double().cpu().view(-1, H + 2 * G, d).split([H, G, G], 1)
    q, k = (O.rotated(O.normed(x, w, c.norm_eps), pos, inv, c.rope_dim, c.rope_style == "neox", mscale) for x, w in ((q, L.q_norm), (k, L.k_norm)))
    kc, vc = ([t[s].cpu() for t in (x.codes, x.scale)] for x, s in zip(eng.cache4[i], (slice(None), slice(None))))
    at = (slots.cpu().long(), slice(None), pos.cpu().long())
    O.assert_held(k, kc[0][at], kc[1][at], 32 * 2.0 ** -24)       # as in the append's own test
    O.assert_held(v, vc[0][at], vc[1][at], 0.0)
    for s in slots.unique().tolist():
        rows = (slots.cpu() == s).nonzero().view(-1)
        p = pos.cpu()[rows]
        n = int(p.max()) + 1
        keys, vals = O.held(kc[0][s, :, :n], kc[1][s, :, :n]), O.held(vc[0][s, :, :n], vc[1][s, :, :n])
        want, err = O.attend(q[rows], keys, vals, p, scale=c.scale, window=c.sliding_window if c.layer_is_swa(i) else 0, softcap=c.attn_softcap,
                             sinks=None if L.sinks is None else L.sinks.cpu(), wide=wide + 2.0 ** -18)      # (2^-18: queries in 32 bits)
        O.assert_near(out.cpu()[rows], want, err)


@pytest.mark.parametrize("spec,ft", [("tiny-qwen3", "Q4_K_M"), ("tiny-qwen2", "Q8_0"), ("tiny-gemma3", "Q8_0"), ("tiny-gemma2", "F16"), ("tiny-tp", "Q4_K_M"), ("sinks", "MXFP4")])
def test_every_layer_against_64_bits(tmp_path, spec, ft, monkeypatch):
    """Prompts of one and of two sequences and steps; windows, local angles, soft caps, norms, sinks and scaled angles as the model has them.  The bounds are the operators' own."""
    from ollama_b200.models.synth import SPECS
    monkeypatch.setitem(SPECS, "sinks", dataclasses.replace(SPECS["tiny-gpt-oss"], head_dim=64))
    _, eng = build(tmp_path, spec, ft)
    eng.alloc(3, 256)
    assert eng.kv_type == "int4"
    eng._pass, eng.use_graphs, seen = None, False, set()      # (the native pass has the same bits: test_int4_engine_gpu.py)
    rows4, step4 = eng._attn_rows4, eng._attn_step4

    def rows(qkv, pos, slots, i, *more):
        o = rows4(qkv, pos, slots, i, *more)
        assert_layer(eng, i, qkv, pos, slots, o, O.HALF16)
        seen.add(("rows", i))
        return o

    def step(i, L, nb):
        step4(i, L, nb)
        b = eng.buf
        assert_layer(eng, i, b.qkv[:nb], b.positions[:nb], b.slots[:nb], b.ao[:nb], 0.0)
        seen.add(("step", i))
    monkeypatch.setattr(eng, "_attn_rows4", rows)
    monkeypatch.setattr(eng, "_attn_step4", step)
    t = tokens(200, 5)
    eng.prefill(1, t[:70], 0)
    eng.prefill_many([(1, t[70:100], 70), (2, t[:37], 0)], [True, True])
    for j in range(3):
        eng.decode([2, 1], [t[100 + j], t[150 + j]], [37 + j, 100 + j])
    eng.decode([0], [t[0]], [0])
    assert seen == {(w, i) for w in ("rows", "step") for i in range(len(eng.layers))} and status() == 0
    eng.close()


@pytest.mark.parametrize("swa", [[True, True], [True, False], [False, True]])
@pytest.mark.parametrize("ft,rows", [("Q4_K_M", 40), ("BF16", 90)])
def test_windows_in_the_native_pass(tmp_path, swa, ft, rows, four_bits):  # noqa: F811
    """Dense layers with a window, alone and beside layers without one, in passes launched from native code: of unit-ordered matrices and of 16-bit ones, of one and of two sequences."""
    from ollama_b200.engine.b200 import B200Backend
    ref, plain = build(tmp_path, "tiny-qwen3", ft, keep_bf16=True)
    plain.close()
    from ollama_b200.engine.backend import open_model
    cfg = dataclasses.replace(ref.cfg, sliding_window=24, swa_layers=swa)
    ref.cfg = ref.model.cfg = cfg
    eng = B200Backend(open_model(str(tmp_path / "m.gguf")), "cuda", kv_type="int4", keep_bf16=True, cfg=cfg)
    near = Near(four_bits)
    for b in (ref, eng):
        b.alloc(2, 256)
    assert eng._pass is not None and eng._pass.windows == {24 if s else 0 for s in swa}
    t = tokens(3 * rows, rows)
    near(eng.verify(0, t[:rows], 0), lambda: ref.verify(0, t[:rows], 0))
    near(eng.verify(0, t[rows:2 * rows - 3], rows), lambda: ref.verify(0, t[rows:2 * rows - 3], rows))
    segs = [(0, t[rows:rows + 20], 2 * rows - 3), (1, t[:rows // 2], 0)]
    got = eng.prefill_many(segs, [True, True])
    for r, a in enumerate(got):
        near(a, lambda: ref.prefill_many(segs, [True, True])[r])
    # other passes launch the same attention
    kept = [x.clone() for x in eng.k_cache + eng.v_cache]
    eng._pass = None
    if ft == "BF16":
        again = eng.prefill_many(segs, [True, True])
        assert all(torch.equal(a, b) for a, b in zip(got, again)) and all(torch.equal(a, b) for a, b in zip(kept, eng.k_cache + eng.v_cache))
    assert status() == 0
    eng.close()


@pytest.mark.parametrize("kv_type", ["f16", "int4"])
def test_passes_count_the_same_launches(tmp_path, kv_type):
    """A pass launched from native code and the same pass launched one by one."""
    from ollama_b200.engine.b200 import B200Backend
    from ollama_b200.engine.backend import open_model
    from ollama_b200.models.synth import write_synthetic_gguf
    p = str(tmp_path / "m.gguf")
    write_synthetic_gguf(p, "tiny-qwen3", "BF16")
    eng, t = B200Backend(open_model(p), "cuda", kv_type=kv_type, keep_bf16=True), tokens(130, 2)
    for segs in ([(0, t[:100], 0)], [(0, t[:80], 100), (1, t[:50], 0)]):
        counts = []
        for native in (True, False):
            eng.alloc(2, 256)
            assert eng._pass.wide
            if not native:
                eng._pass = None
            before = eng.kernel_launches
            eng._forward_rows(segs)
            counts.append(eng.kernel_launches - before)
        assert counts[0] == counts[1], (segs, counts)
    eng.close()


def test_served_tokens_are_those_of_each_sequence(tmp_path):
    """Requests that arrive together and share a prefix, 40 steps each: every token is one that the sequence alone might have been given.  Engine and graph differ by up to 5 % of the largest logit and what
    four bits move it by (test_int4_engine_gpu.py), so the logits of two engines by twice that, D, and a token of the largest served logit is within 2 D of the largest of the sequence alone."""
    from ollama_b200.engine.b200 import B200Backend
    from ollama_b200.engine.backend import open_model
    from ollama_b200.engine.runner import CompletionRequest, Runner, RunnerOptions
    from ollama_b200.engine.sampler import SamplingParams
    from ollama_b200.models.synth import write_synthetic_gguf
    p = str(tmp_path / "m.gguf")
    write_synthetic_gguf(p, "tiny-qwen3", "Q8_0")
    prompt = tokens(100, 3)
    prompts = [prompt, prompt[:80] + prompt[:9], prompt[::-1], tokens(60, 9)]
    r = Runner(p, RunnerOptions(num_ctx=256, num_parallel=4, num_batch=48, device="cuda", kv_cache_type="int4"))
    served = []
    try:
        for a in [r.submit(CompletionRequest(prompt=list(x), sampling=SamplingParams(temperature=0), num_predict=40, ignore_eos=True)) for x in prompts]:
            got, done = [], False
            while not done:
                c = a.out.get(timeout=60)
                got += c.tokens
                done = c.done
            served.append(got)
    finally:
        r.close()
    four, sixteen = (B200Backend(open_model(p), "cuda", kv_type=t) for t in ("int4", "f16"))
    for e in (four, sixteen):
        e.alloc(1, 256)
    for x, got in zip(prompts, served):
        assert len(got) == 40
        rows = []
        for e in (four, sixteen):
            rows.append([e.prefill(0, x, 0).float().cpu()] + [e.decode([0], [t], [len(x) + j])[0].float().cpu() for j, t in enumerate(got[:-1])])
        for t, a, b in zip(got, *rows):
            d = 2 * (0.05 * a.abs().max() + (a - b).abs().max())
            assert a[t] >= a.max() - 2 * d, (t, float(a[t]), float(a.max()), float(d))
    for e in (four, sixteen):
        e.close()


def test_a_bench_line_says_what_the_cache_holds(tmp_path):
    import bench
    from ollama_b200.engine.b200 import B200Backend
    from ollama_b200.engine.backend import open_model
    from ollama_b200.models.synth import write_synthetic_gguf
    for spec, ft, holds in (("tiny-gpt-oss", "MXFP4", "q8_0"), ("tiny-qwen3", "Q8_0", "int4")):
        p = str(tmp_path / f"{spec}.gguf")
        write_synthetic_gguf(p, spec, ft)
        eng = B200Backend(open_model(p), "cuda", kv_type="int4")
        assert bench.kv_cache(eng) == holds
        eng.close()
