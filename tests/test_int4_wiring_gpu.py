"""Models under OLLAMA_KV_CACHE_TYPE=int4: launches of passes, what a bench line says of the cache."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def tokens(n, seed):
    return torch.randint(259, 4096, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


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
