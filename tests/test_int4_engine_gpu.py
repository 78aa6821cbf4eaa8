"""Models under OLLAMA_KV_CACHE_TYPE=int4, against the fp32 graph whose attention sees keys and values as a 4-bit cache holds them."""
import logging

import pytest
import torch

import kv4_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture
def four_bits(monkeypatch):
    """Switches the fp32 graph's rounding on and off."""
    from ollama_b200.models import reference
    real, state = reference.R.attention, {"on": True}

    def attention(q, k, v, *a, **kw):
        if state["on"]:
            k, v = (O.rounded(x.double()).to(torch.float16).float() for x in (k, v))
        return real(q, k, v, *a, **kw)
    monkeypatch.setattr(reference.R, "attention", attention)
    return state


def build(tmp_path, spec, ft, **kw):
    from ollama_b200.engine.b200 import B200Backend
    from ollama_b200.engine.backend import TorchBackend, open_model
    from ollama_b200.models.synth import write_synthetic_gguf
    p = str(tmp_path / "m.gguf")
    write_synthetic_gguf(p, spec, ft)
    return TorchBackend(open_model(p), "cpu"), B200Backend(open_model(p), "cuda", kv_type="int4", **kw)


def status():
    from ollama_b200.ops import cuda as K
    return K.gemm_status()


class Near:
    """The engine rounds the inputs of products to 16 bits or less (5 % of the largest logit, the bound of the whole-model tests), and moves codes near a border by a step: at most as much again as
    rounding to four bits moves the logits, since a step is twice the largest rounding and a code in a few is that near."""

    def __init__(self, state):
        self.state = state

    def __call__(self, got, ask):
        """``ask()``: the graph's logits; asked twice, with and without the rounding (it writes the same cache)."""
        self.state["on"] = False
        plain = ask()
        self.state["on"] = True
        want = ask()
        off = (got.float().cpu() - want).abs().max().item()
        assert off < 0.05 * want.abs().max().item() + (want - plain).abs().max().item(), off
        return want


@pytest.mark.parametrize("spec,ft", [("tiny-qwen3", "Q4_K_M"), ("tiny-qwen3", "Q8_0"), ("tiny-gemma3", "Q8_0"), ("tiny-gemma2", "F16"), ("tiny-qwen3moe", "Q8_0"), ("tiny-tp", "Q4_K_M")])
def test_prompts_and_steps(tmp_path, spec, ft, four_bits):
    ref, eng = build(tmp_path, spec, ft)
    near = Near(four_bits)
    for b in (ref, eng):
        b.alloc(3, 256)
    assert eng.kv_type == "int4" and eng.kv_bytes() == sum(2 * t.numel() // 2 + 2 * t.numel() // 32 * 2 for t in ref.cache.k)
    prompt = torch.randint(259, 4096, (150,), generator=torch.Generator().manual_seed(3)).tolist()
    near(eng.prefill(1, prompt[:70], 0), lambda: ref.prefill(1, prompt[:70], 0))
    near(eng.prefill(1, prompt[70:], 70), lambda: ref.prefill(1, prompt[70:], 70))
    near(eng.verify(1, prompt[:5], 150), lambda: ref.verify(1, prompt[:5], 150))
    segs = [(0, prompt[:33], 0), (2, prompt[40:], 0)]
    wants = []
    for r, a in enumerate(eng.prefill_many(segs, [True, True])):
        wants.append(near(a, lambda: ref.prefill_many(segs, [True, True])[r]))
    toks, pos = [int(w.argmax()) for w in wants], [33, 110]
    for step in range(4):          # the second call is the captured step
        got = eng.decode([0, 2], toks, pos)
        if ref.cfg.is_moe:           # a near tie of the router's turns where a key's code does, and the logits with it: against the prompt pass, which finds the same cache
            want = torch.cat([eng.verify(s, [t], p) for s, t, p in zip((0, 2), toks, pos)])
            assert (got - want).abs().max() < 0.05 * want.abs().max()
            toks, pos = want.argmax(-1).tolist(), [p + 1 for p in pos]
            continue
        want = near(got, lambda: torch.stack([ref.decode([s], [t], [p])[0] for s, t, p in zip((0, 2), toks, pos)]))
        toks, pos = want.argmax(-1).tolist(), [p + 1 for p in pos]
    assert status() == 0
    eng.check_waits()
    eng.close()


@pytest.mark.parametrize("rows", [1, 64, 65])
@pytest.mark.parametrize("ft", ["Q4_K_M", "BF16"])
def test_native_prompt_pass(tmp_path, rows, ft, four_bits):
    """Passes launched from native code, on both sides of the rows up to which they read unit-ordered matrices, and of two sequences."""
    ref, eng = build(tmp_path, "tiny-qwen3", ft, keep_bf16=True)
    near = Near(four_bits)
    for b in (ref, eng):
        b.alloc(2, 256)
    assert eng._pass is not None and eng._pass.wide and eng._pass.units == (ft == "Q4_K_M")
    prompt = torch.randint(259, 4096, (2 * rows,), generator=torch.Generator().manual_seed(rows)).tolist()
    near(eng.verify(0, prompt[:rows], 0), lambda: ref.verify(0, prompt[:rows], 0))
    near(eng.prefill(0, prompt[rows:], rows), lambda: ref.prefill(0, prompt[rows:], rows))
    segs = [(0, prompt[:rows], 0), (1, prompt[rows:rows + (rows + 1) // 2], 0)]
    for r, a in enumerate(eng.prefill_many(segs, [True, True])):
        near(a, lambda: ref.prefill_many(segs, [True, True])[r])
    assert status() == 0
    eng.close()


def test_a_step_does_not_depend_on_the_pass(tmp_path):
    """Native and other passes launch the same attention: the same cache and logits."""
    ref, eng = build(tmp_path, "tiny-qwen3", "BF16", keep_bf16=True)
    prompt = torch.randint(259, 4096, (90,), generator=torch.Generator().manual_seed(1)).tolist()
    got = []
    for native in (True, False):
        eng.alloc(1, 128)
        if not native:
            eng._pass = None
        logits = eng.prefill(0, prompt, 0)
        got.append((logits, *[t.clone() for t in eng.k_cache + eng.v_cache + eng.k_scale + eng.v_scale]))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    eng.close()


def test_rows_copied_and_shifted(tmp_path, four_bits):
    """A prefix in another slot is the same prefix; dropped rows leave the keys behind them turned back and rounded again."""
    ref, eng = build(tmp_path, "tiny-qwen3", "F16")
    near = Near(four_bits)
    for b in (ref, eng):
        b.alloc(2, 128)
    toks = torch.randint(259, 4096, (90,), generator=torch.Generator().manual_seed(3)).tolist()
    for b in (ref, eng):
        b.prefill(0, toks, 0)
        b.copy_rows(0, 1, 60)
    one = eng.decode([0], [5], [60])
    eng.prefill(0, toks, 0)
    assert torch.equal(one, eng.decode([1], [5], [60]))
    for b in (ref, eng):
        b.prefill(0, toks, 0)
    k0 = [eng.cache4[i][0] for i in range(2)]
    rows = [O.held(k.codes[0, :, 45:90].cpu(), k.scale[0, :, 45:90].cpu()) for k in k0]
    for b in (ref, eng):
        b.shift(0, 5, 40, 90)
    inv = eng.inv_freq.cpu()
    for k, x in zip(k0, rows):
        want = O.rotated(x.transpose(0, 1), torch.full((45,), -40), inv, 64, eng.cfg.rope_style == "neox").transpose(0, 1)
        O.assert_held(want, k.codes[0, :, 5:50], k.scale[0, :, 5:50], 64 * 2.0 ** -24)
    # the graph's rows are rounded once, the engine's twice
    near(eng.decode([0], [toks[-1]], [50])[0], lambda: ref.decode([0], [toks[-1]], [50])[0])
    eng.close()


def test_image_rows(tmp_path, four_bits):
    ref, eng = build(tmp_path, "tiny-gemma3", "F16")
    near = Near(four_bits)
    g = torch.Generator().manual_seed(4)
    toks = torch.randint(259, 4096, (60,), generator=g).tolist()
    rows = list(range(20, 36))
    for r in rows:
        toks[r] = -(1 + r)
    emb, spans = torch.randn(len(rows), ref.cfg.d_model, generator=g) * 0.5, [(20, 36)]
    for e in (ref, eng):
        e.alloc(1, 128)
    near(eng.prefill(0, toks, 0, embeds=(rows, emb.cuda()), spans=spans), lambda: ref.prefill(0, toks, 0, embeds=(rows, emb), spans=spans))
    near(eng.decode([0], [7], [60])[0], lambda: ref.decode([0], [7], [60])[0])
    eng.close()


def test_models_without_four_bits(tmp_path, caplog):
    """Head sizes that the cache does not have are stored as before, and the log says so; other 4-bit names keep what they were."""
    from ollama_b200.engine.b200 import B200Backend
    from ollama_b200.engine.backend import open_model
    from ollama_b200.models.synth import write_synthetic_gguf
    p, r = str(tmp_path / "m.gguf"), str(tmp_path / "n.gguf")
    write_synthetic_gguf(p, "tiny-gpt-oss", "MXFP4")
    write_synthetic_gguf(r, "tiny-qwen3", "Q8_0")
    with caplog.at_level(logging.WARNING, "ollama_b200.engine"):
        assert B200Backend(open_model(p), "cuda", kv_type="int4").kv_type == "q8_0"
        assert B200Backend(open_model(r), "cuda", kv_type="q4_0").kv_type == "q8_0"
    assert [m.getMessage().split(" is stored as ")[0] for m in caplog.records] == ["K/V cache type int4", "K/V cache type q4_0"]


def test_requests_side_by_side(tmp_path):
    """A served model: requests that arrive together and share a prefix answer as each alone does."""
    from ollama_b200.engine.runner import CompletionRequest, Runner, RunnerOptions
    from ollama_b200.engine.sampler import SamplingParams
    from ollama_b200.models.synth import write_synthetic_gguf
    p = str(tmp_path / "m.gguf")
    write_synthetic_gguf(p, "tiny-qwen3", "Q8_0")
    prompt = torch.randint(259, 4096, (100,), generator=torch.Generator().manual_seed(3)).tolist()
    prompts = [prompt, prompt[:80] + prompt[:9], prompt[::-1]]

    def answers(together):
        r = Runner(p, RunnerOptions(num_ctx=256, num_parallel=3, num_batch=48, device="cuda", kv_cache_type="int4"))
        try:
            assert r.backend.kv_type == "int4"
            ask = lambda x: r.submit(CompletionRequest(prompt=list(x), sampling=SamplingParams(temperature=0), num_predict=12, ignore_eos=True))
            got = []
            for group in ([prompts] if together else [[x] for x in prompts]):
                for a in [ask(x) for x in group]:
                    tokens, done = [], False
                    while not done:
                        c = a.out.get(timeout=60)
                        tokens += c.tokens
                        done = c.done
                    got.append(tokens)
            return got
        finally:
            r.close()
    one, both = answers(False), answers(True)
    assert all(len(t) == 12 for t in one + both)
    # sums in another order may turn a near tie, not the first tokens of all
    assert sum(a[0] == b[0] for a, b in zip(one, both)) >= 2
