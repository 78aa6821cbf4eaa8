"""Stack models under OLLAMA_KV_CACHE_TYPE=fp8: models that it does not reach, what a step counts, requests side by side."""
import logging

import pytest
import torch

import kavenex_models as KM
import vazatar_models as VM
from test_fp8_cache_gpu import engine

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
