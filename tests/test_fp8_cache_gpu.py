"""Stack models on the 8-bit cache: logits against the plain implementation with keys and values rounded as the cache rounds them, however the tokens are cut into steps,
batched, placed in slots, or generated."""
import pytest
import torch

import pages8_oracle as P8
import rinirax_models as RM
import rinirax_oracle as RO
import tirudra_models as TM
import tirudra_oracle as TO
import vazatar_models as VM
import vazatar_oracle as VO
from test_vazatar_gpu import errors, run

pytestmark = pytest.mark.gpu

CONFIGS = {
    "vazatar-small": (VM, VM.small()),
    "vazatar-wide": (VM, VM.config([VM.attention(heads=20, kv_heads=1, dim=96, vdim=128, size=130, rot={"base": 1e4, "dims": 96}), VM.mamba(inner=60, state=20, dt_rank=5, conv=3),
                                    VM.attention(heads=4, kv_heads=2, dim=128, vdim=72, size=96, scale=0.1, rot={"base": 1e4, "dims": 64}, softcap=0.0)], width=136, vocab=301,
                                   loop=(0, 3, 2), cap=0.0)),
    "vazatar-heads": (VM, VM.config([VM.attention(), VM.attention(heads=4, kv_heads=2, dim=24, vdim=24, size=64, rot={"base": 90.0, "dims": 24}), VM.attention(size=0)], loop=None)),
    "tirudra-plain": (TM, TM.config([TM.windowed(), TM.mamba(), TM.full(), TM.windowed(heads=8, kv_heads=2, dim=64, vdim=64, size=100, keep=70), TM.full(heads=8, kv_heads=2, dim=128)])),
    "rinirax-plain": (RM, RM.config([RM.diff(RM.dense(), heads=6, kv_heads=2, dim=32, vdim=64, scale=0.2), RM.gru(RM.dense(9)), RM.latent(RM.dense(70), size=100),
                                     RM.diff(kv_from=0, heads=6, kv_heads=2, dim=32, vdim=64, conv=2), RM.diff(RM.dense(30), heads=8, kv_heads=1, dim=64, vdim=128, conv=2, scale=0.12)])),
}
ORACLES = {VM: VO, TM: TO, RM: RO}


def held(x):
    """Rows [T, kv heads, columns] as pages of the cache hold them when they are full."""
    out = []
    for p in range(0, len(x), 64):
        y = x[p:p + 64].transpose(0, 1)
        u = P8.unit_for(y.abs().amax((1, 2)))[:, None, None]
        out.append((P8.e4m3(y / u) * u).transpose(0, 1))
    return torch.cat(out)


@pytest.fixture
def rounded_caches(monkeypatch):
    def around(f):
        return lambda q, k, v, *a: f(q, held(k), held(v), *a)

    def keys_values(f):
        def call(*a):
            k, v = f(*a)
            return held(k.flatten(2)).view(k.shape), held(v)
        return call
    monkeypatch.setattr(VO, "attend", around(VO.attend))
    monkeypatch.setattr(TO, "attend", around(TO.attend))
    monkeypatch.setattr(RO, "keys_values", keys_values(RO.keys_values))


def engine(path, dtype="bfloat16", slots=4, ctx=512, kv="fp8"):
    from ollama_b200.engine.backend import make_backend, open_model
    from ollama_b200.engine.runner import RunnerOptions
    with open_model(path) as g:
        be = make_backend(g, "cuda", opts=RunnerOptions(dtype=dtype, kv_cache_type=kv))
    be.alloc(slots, ctx)
    return be


@pytest.mark.parametrize("name", list(CONFIGS))
def test_logits(name, tmp_path, rounded_caches):
    """Bound as for 16-bit caches: what rounding the products' inputs to bf16 does to the logits, here through the cache's codes too, times three."""
    from ollama_b200.ops import cuda as K
    M, cfg = CONFIGS[name]
    O = ORACLES[M]
    w = M.weights(cfg, len(name))
    be = engine(M.write(tmp_path, cfg, w))
    assert be.fp8
    toks, more = M.tokens(203, cfg["vocab"], 7), M.tokens(90, cfg["vocab"], 9)
    want, want2 = O.forward(cfg, w, toks), O.forward(cfg, w, more)
    base = errors(O.forward(cfg, w, toks, product=O.rounded), want).max()
    base2 = errors(O.forward(cfg, w, more, product=O.rounded), want2).max()

    def check(got, want, base, note):
        e = errors(got, want)
        assert torch.isfinite(got).all() and e.max() < 3 * base, (note, float(e.max()), float(base))
    for slot, cuts in enumerate([[203], [1], [2], [3, 61, 64, 2, 5, 1, 1, 30]]):
        check(run(be, slot, toks, cuts), want, base, cuts)
    # two sequences side by side, portions beside single tokens, in slots that others have used
    got, at = [[], []], [0, 0]
    for n in ((100, 40), (1, 1), (63, 1), (1, 30), (1, 1), (37, 17)):
        out = be.step([(3, toks[at[0]:at[0] + n[0]], at[0]), (1, more[at[1]:at[1] + n[1]], at[1])], [range(n[0]), range(n[1])])
        got[0].append(out[:n[0]])
        got[1].append(out[n[0]:])
        at = [a + k for a, k in zip(at, n)]
    check(torch.cat(got[0]), want, base, "beside")
    check(torch.cat(got[1]), want2, base2, "beside")
    if not be.cfg.recurrent:
        be.copy_rows(3, 0, 150)
        check(be.step([(0, toks[150:203], 150)], [range(53)]), want[150:], base, "a prefix of another slot")
        be.free_slot(0)
    assert K.gemm_status() == 0
    be.close()


def test_captured_loop_equals_single_steps(tmp_path):
    M, cfg = CONFIGS["vazatar-small"]
    w = M.weights(cfg, 3)
    be = engine(M.write(tmp_path, cfg, w))
    toks = M.tokens(70, cfg["vocab"], 5)
    for s in (0, 1):
        be.step([(s, toks[:50 + 10 * s], 0)], [[]])
    first = [5, 6]
    loop = be.decode_loop([0, 1], first, [50, 60], 24).cpu().tolist()
    for s in (0, 1):
        be.free_slot(s)
        be.step([(s, toks[:50 + 10 * s], 0)], [[]])
    cur, at = first, [50, 60]
    for row in loop:
        cur = be.decode([0, 1], cur, at).argmax(-1).tolist()
        assert cur == row
        at = [a + 1 for a in at]
    be.close()


def test_which_layers_and_models_have_it(tmp_path):
    """Half the bytes; wide heads, latents and 32-bit models keep their caches; other names of types keep theirs too."""
    M, cfg = CONFIGS["tirudra-plain"]
    w = M.weights(cfg, 3)
    path = M.write(tmp_path / "a", cfg, w) if (tmp_path / "a").mkdir() is None else None
    sizes = {}
    for kv, dtype, fp8 in (("f16", "bfloat16", False), ("fp8", "bfloat16", True), ("q8_0", "bfloat16", False), ("fp8", "float32", False)):
        be = engine(path, dtype, kv=kv)
        assert be.fp8 == fp8
        sizes[kv, dtype] = sum(t.numel() * t.element_size() for t in be.cache.paged)
        be.close()
    assert sizes["q8_0", "bfloat16"] == sizes["f16", "bfloat16"] and sizes["fp8", "bfloat16"] < 0.51 * sizes["f16", "bfloat16"]
    wide = VM.config([VM.attention(heads=2, kv_heads=1, dim=160, vdim=200, size=0, rot={}, scale=0.05, ff=33), VM.attention(heads=2, kv_heads=1, dim=16, vdim=20)], width=37, vocab=59, loop=None)
    (tmp_path / "b").mkdir()
    w = VM.weights(wide, 4)
    be = engine(VM.write(tmp_path / "b", wide, w))
    assert torch.isfinite(run(be, 0, VM.tokens(90, 59, 1), [80, 1])).all()
    assert [isinstance(m[0], torch.Tensor) for m in be.mem] == [True, False]
    be.close()


def test_two_portions_of_one_slot_are_refused(tmp_path):
    M, cfg = CONFIGS["vazatar-small"]
    w = M.weights(cfg, 3)
    be = engine(M.write(tmp_path, cfg, w))
    with pytest.raises(ValueError, match="one slot"):
        be.step([(1, [3, 4], 0), (1, [5, 6], 2)], [[], []])
    be.close()


def test_generation_through_the_runner(tmp_path):
    """Two requests at once, one behind the other's prefix, as a server runs them."""
    from ollama_b200.engine.runner import CompletionRequest, Runner, RunnerOptions
    from ollama_b200.engine.sampler import SamplingParams
    M, cfg = CONFIGS["vazatar-small"]
    w = M.weights(cfg, 3)
    path = M.write(tmp_path, cfg, w)
    r = Runner(str(path), RunnerOptions(num_ctx=256, num_parallel=2, device="cuda", kv_cache_type="fp8"))
    try:
        assert r.backend.fp8
        prompt = M.tokens(100, cfg["vocab"], 4)
        outs = []
        for p in (prompt, prompt[:80] + M.tokens(9, cfg["vocab"], 8), prompt):
            outs.append([t for c in r.completion(CompletionRequest(prompt=list(p), sampling=SamplingParams(temperature=0), num_predict=12, ignore_eos=True)) for t in c.tokens])
        assert all(len(o) == 12 for o in outs)
    finally:
        r.close()
