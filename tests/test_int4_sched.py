"""What the scheduler counts for models under OLLAMA_KV_CACHE_TYPE=int4: four bits where the model comes to one GPU, eight where ranks that share it keep int8."""
from types import SimpleNamespace

import pytest

from ollama_b200.discover.devices import DeviceInfo
from ollama_b200.server.sched import Scheduler, predict_memory

GB = 10 ** 9
TOKEN = 2 * 32 * 8 * 128                       # cached values of a token
COPY = 2 * (32 * (4096 * (2 * 4096 + 2 * 1024) + 3 * 4096 * 14336) + 128256 * 4096)


@pytest.fixture
def model(monkeypatch):
    monkeypatch.setenv("OLLAMA_KV_CACHE_TYPE", "int4")
    for n in ("OLLAMA_SCHED_SPREAD", "B200_TP"):
        monkeypatch.delenv(n, raising=False)
    kv = {"block_count": 32, "attention.head_count": 32, "attention.head_count_kv": 8, "embedding_length": 4096, "feed_forward_length": 14336, "vocab_size": 128256}
    kv = {"general.architecture": "llama"} | {f"llama.{n}": v for n, v in kv.items()}
    return SimpleNamespace(size=5 * GB, kv=lambda: kv)


def four(ctx, n):
    return 5 * GB + TOKEN * ctx * n * 9 // 16


def eight(ctx, n):
    return 5 * GB + TOKEN * ctx * n * 34 // 32 + 2 * 8 * 128 * ctx * 2


def gpus(n, free):
    return [DeviceInfo(id=str(i), index=i, total_memory=free, free_memory=free) for i in range(n)]


def test_the_prefill_copy_counts_where_the_choice_is_made(model):
    """The cache alone fits 80 % of a GPU, beside the 16-bit copy of the matrices it does not: the model goes to two GPUs, whose ranks keep int8."""
    free, ctx, n = 100 * GB, 131072, 14
    assert four(ctx, n) < 0.8 * free < four(ctx, n) + COPY and COPY < 0.4 * free
    need = predict_memory(model, ctx, n, free=free)
    assert need == eight(ctx, n) + COPY
    assert len(Scheduler._place(gpus(2, free), need)) == 2


def test_four_bits_are_counted_where_one_gpu_takes_the_model(model):
    """Over sizes on both sides of every limit, on two GPUs: a prediction of four bits and a placement on one GPU go together."""
    for free in (30 * GB, 60 * GB, 100 * GB, 180 * GB):
        for n in range(1, 40):
            ctx = 40960
            need, copy = predict_memory(model, ctx, n, free=free), COPY if COPY < 0.4 * free else 0
            assert need in (four(ctx, n) + copy, eight(ctx, n) + copy)
            assert (len(Scheduler._place(gpus(2, free), need)) == 1) == (need == four(ctx, n) + copy), (free, n)


@pytest.mark.parametrize("name", ["B200_TP", "OLLAMA_SCHED_SPREAD"])
def test_forced_groups_keep_int8(model, monkeypatch, name):
    assert predict_memory(model, 4096, 2, free=180 * GB) == four(4096, 2) + COPY
    monkeypatch.setenv(name, "2" if name == "B200_TP" else "1")
    assert predict_memory(model, 4096, 2, free=180 * GB) == eight(4096, 2) + COPY
    assert predict_memory(model, 4096, 2) == eight(4096, 2)


@pytest.mark.parametrize("name", ["", "B200_TP", "OLLAMA_SCHED_SPREAD"])
def test_a_node_of_one_gpu_has_no_groups(model, monkeypatch, name):
    """Its runner keeps four bits however little is left beside the cache, so an automatic context is not cut as if it were eight."""
    if name:
        monkeypatch.setenv(name, "2" if name == "B200_TP" else "1")
    free, ctx, n = 180 * GB, 262144, 15
    assert 0.8 * free < four(ctx, n) + COPY < free < eight(ctx, n) + COPY
    assert predict_memory(model, ctx, n, free=free, gpus=1) == four(ctx, n) + COPY
    assert predict_memory(model, ctx, n, free=free, gpus=2) == eight(ctx, n) + COPY
    seen = []
    s = Scheduler(new_runner_fn=lambda m, opts, parallel, use: (seen.append((opts["num_ctx"], len(use))), SimpleNamespace(close=lambda: None, ping=lambda: True))[1], get_gpus_fn=lambda: gpus(1, free))
    monkeypatch.setenv("OLLAMA_NUM_PARALLEL", str(n))
    model.model_path, model.name = "/blobs/a", "a"
    s.release(s.get_runner(model, {"num_ctx": 0}, 60))
    s.unload_all()
    assert seen == [(ctx, 1)]
