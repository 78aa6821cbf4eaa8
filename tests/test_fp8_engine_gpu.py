"""Stack models under OLLAMA_KV_CACHE_TYPE=fp8: models that it does not reach, what a step counts, requests side by side."""
import logging

import pytest
import torch

import kavenex_models as KM
import vazatar_models as VM
import vazatar_oracle as VO
from test_fp8_cache_gpu import CONFIGS, engine, rounded_caches  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("model", ["latents", "wide"])
def test_models_without_8_bit_pages_run_as_they_did(model, tmp_path, caplog):
    """Latent rows and wide heads stay in 16 bits: a step of two portions of one slot is taken, its results are those of the other cache type, and the log says that nothing changed."""
    if model == "latents":
        M, cfg = KM, KM.config([KM.layer(KM.dense()), KM.layer(), KM.layer(KM.dense(40))])
    else:
        M, cfg = VM, VM.config([VM.attention(heads=2, kv_heads=1, dim=160, vdim=200, size=0, rot={}, scale=0.05, ff=33)], width=37, vocab=59, loop=None)
    path = M.write(tmp_path, cfg, M.weights(cfg, 3))
    toks, got = M.tokens(20, cfg["vocab"], 5), []
    for kv in ("f16", "fp8"):
        with caplog.at_level(logging.WARNING, "ollama_b200.engine"):
            be = engine(path, kv=kv)
        got.append(be.step([(1, toks[:12], 0), (1, toks[12:], 12)], [range(12), range(8)]))
        be.close()
    assert torch.equal(*got)
    assert [r.getMessage().split(":")[0] for r in caplog.records] == ["K/V cache type fp8 changes nothing"]


def test_other_models_refuse_the_type(tmp_path):
    """A model whose engine has no E4M3 cache does not get another 8-bit one in its place."""
    from ollama_b200.engine.b200 import B200Backend
    from ollama_b200.engine.backend import open_model
    from ollama_b200.models.synth import write_synthetic_gguf
    path = str(tmp_path / "m.gguf")
    write_synthetic_gguf(path, "tiny-qwen3", "Q8_0")
    for kv, what in (("fp8", "stack models"), ("fp9", "unknown")):
        with pytest.raises(ValueError, match=what), open_model(path) as g:
            B200Backend(g, "cuda", kv_type=kv)


def test_a_step_counts_what_it_copies(tmp_path):
    """A mixed step brings its rows, its portions and, once for each mask, what the 8-bit attention has to know of them to the device."""
    cfg = VM.config([VM.attention(), VM.attention(size=96), VM.attention()], loop=None)
    path = VM.write(tmp_path, cfg, VM.weights(cfg, 3))
    got = {}
    for kv in ("f16", "fp8"):
        be = engine(path, kv=kv)
        be.step([(0, VM.tokens(20, cfg["vocab"], 5), 0)], [[]])
        before = be.h2d_bytes
        be.step([(0, VM.tokens(70, cfg["vocab"], 6), 20), (2, [3], 0)], [[], []])
        got[kv] = be.h2d_bytes - before
        chunks = {L.mixer.chunk for L in be.layers}
        if kv == "fp8":
            from ollama_b200.ops import pages8 as P
            plans = [P.portions8([(0, 70, 0, 20), (70, 1, 2, 0)], be.cache.table, chunk=c).nbytes for c in chunks]
        be.close()
    assert len(plans) == 2 and got["fp8"] == got["f16"] + sum(plans)


def test_requests_side_by_side(tmp_path, rounded_caches):
    """A request is generating while others arrive, one with most of its prompt: portions beside single tokens, a prefix copied out of a busy slot.  Every token has the largest logit
    of the plain implementation on rounded caches, or one nearer to it than twice what rounding the products' inputs does to a logit, times three as in test_logits."""
    from ollama_b200.engine.runner import CompletionRequest, Runner, RunnerOptions
    from ollama_b200.engine.sampler import SamplingParams
    cfg = CONFIGS["vazatar-heads"][1]
    w = VM.weights(cfg, 3)
    r = Runner(str(VM.write(tmp_path, cfg, w)), RunnerOptions(num_ctx=320, num_parallel=3, num_batch=48, device="cuda", kv_cache_type="fp8"))
    prompt = VM.tokens(100, cfg["vocab"], 4)
    prompts = [prompt, prompt[:80] + VM.tokens(9, cfg["vocab"], 8), VM.tokens(130, cfg["vocab"], 11)]

    def request(p, n):
        return r.submit(CompletionRequest(prompt=list(p), sampling=SamplingParams(temperature=0), num_predict=n, ignore_eos=True))
    try:
        assert r.backend.pages8
        asked = [request(prompts[0], 120)]
        got = [asked[0].out.get(timeout=60).tokens]                     # its prompt is in the cache and it is generating
        asked += [request(p, 20) for p in prompts[1:]]
        got += [[], []]
        for a, tokens in zip(asked, got):
            done = False
            while not done:
                c = a.out.get(timeout=60)
                tokens += c.tokens
                done = c.done
        assert [len(t) for t in got] == [120, 20, 20] and r.stats["mixed_steps"] > 0 and r.stats["prefix_copies"] > 0
    finally:
        r.close()
    for p, tokens in zip(prompts, got):
        rows = list(p) + tokens[:-1]
        want, near = VO.forward(cfg, w, rows), VO.forward(cfg, w, rows, product=VO.rounded)
        logits = want[len(p) - 1:].cpu()
        behind = logits.amax(-1) - logits[torch.arange(len(tokens)), torch.tensor(tokens)]
        assert behind.max() <= 2 * 3 * (near - want).abs().max(), float(behind.max())
