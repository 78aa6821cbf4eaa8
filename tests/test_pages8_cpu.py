"""The 8-bit paged cache's host side: which portions and tensors are refused."""
import pytest
import torch

import pages8_oracle as O
from ollama_b200.ops import pages8 as P

TABLE = torch.zeros(3, 4, dtype=torch.int32)


def test_portions():
    p = P.portions8([(0, 5, 2, 62), (5, 130, 0, 0), (135, 1, 1, 255)], TABLE)
    assert p.rows == 136 and p.per == 3 and p.longest == 130 and p.segs.tolist() == [[0, 5, 2, 62], [5, 130, 0, 0], [135, 1, 1, 255]]


def test_pages_that_portions_see():
    table = torch.zeros(2, 20, dtype=torch.int32)
    p = P.portions8([(0, 130, 1, 700), (130, 3, 0, 0)], table, window=200, keep=70)
    # keys from 501 on, in tiles of 128 from 384 (page 6) on, to 829 (page 12), and the kept ones in the first tile
    assert p.pages.tolist() == [[1, b, 64, 0] for b in (0, 1, 6, 7, 8, 9, 10, 11)] + [[1, 12, 62, 0], [0, 0, 3, 0]]
    assert p.table[0, [0, 1, 6, 12]].tolist() == [0, 1, 2, 8] and p.table[1, 0] == 9
    assert p.tiles.tolist() == [[0, 128, 0, 700], [128, 2, 0, 828], [130, 3, 1, 0]] and p.half_tiles.tolist()[2] == [128, 2, 0, 828]
    assert P.portions8([(0, 2, 0, 300)], table, chunk=150).pages.tolist() == [[0, 4, 46, 0]]
    for mask in (dict(window=-1), dict(keep=-1), dict(chunk=-3), dict(chunk=3, window=5)):
        with pytest.raises(ValueError):
            P.portions8([(0, 2, 0, 300)], table, **mask)


@pytest.mark.parametrize("parts", [[], [(0, 0, 0, 0)], [(1, 3, 0, 0)], [(0, 3, 0, 0), (2, 3, 1, 0)], [(0, 3, 0, 0), (4, 3, 1, 0)], [(0, 3, 3, 0)], [(0, 3, -1, 0)], [(0, 3, 0, -1)],
                                   [(0, 3, 0, 254)], [(0, 1, 0, 256)], [(0, 3, 0, 0), (3, 3, 0, 3)]])
def test_portions_that_are_refused(parts):
    with pytest.raises(ValueError):
        P.portions8(parts, TABLE)


def test_pages_that_are_refused():
    ok = torch.zeros(2, 3, 64, 64, dtype=torch.uint8)
    P.Pages8(ok, torch.ones(2, 3))
    for codes, unit in ((ok.float(), torch.ones(2, 3)), (ok[:, :, :32], torch.ones(2, 3)), (ok.transpose(0, 1), torch.ones(3, 2)), (ok, torch.ones(2, 4)), (ok, torch.ones(2, 3).half()),
                        (torch.zeros(2, 3, 64, 96, dtype=torch.uint8), torch.ones(2, 3)), (ok[0], torch.ones(2, 3))):
        with pytest.raises(ValueError):
            P.Pages8(codes, unit)
    for dim in (0, 129):
        with pytest.raises(ValueError):
            P.Pages8.empty(2, 3, dim, device="cpu")


def test_calls_on_the_cpu_are_refused():
    k, v = P.Pages8.empty(2, 1, 64, device="cpu"), P.Pages8.empty(2, 1, 64, device="cpu")
    x, q, i = torch.zeros(1, 192), torch.zeros(1, 1, 64), torch.zeros(1, dtype=torch.int32)
    prep = dict(heads=1, dim=64, vdim=64, q_norm=None, k_norm=None, eps=1e-5, freqs=None, n_rot=0)
    with pytest.raises(ValueError, match="cpu"):
        P.append8(x, k, v, TABLE, q, positions=i, slots=i, **prep)
    with pytest.raises(ValueError, match="cpu"):
        P.attn_decode8(x, k, v, i, i, TABLE, torch.zeros(1, 64), n_ctx=64, scale=1.0, **prep)
    with pytest.raises(ValueError, match="cpu"):
        P.attn_prompt8(q, k, v, P.portions8([(0, 1, 0, 0)], TABLE), TABLE, torch.zeros(1, 64), vdim=64, scale=1.0)
    with pytest.raises(ValueError, match="cpu"):
        P.read8(k, v, torch.zeros(1, 4, dtype=torch.int32), TABLE, torch.zeros(1, 1, 64, 64), torch.zeros(1, 1, 64, 64))


def test_the_definition():
    """The oracle's rounding is the type's, and its units hold the largest magnitude."""
    x = torch.cat([torch.arange(-448, 449).double() / 3, torch.randn(4000, generator=torch.Generator().manual_seed(1)).double() * 0.01])
    assert torch.equal(O.e4m3(x), x.float().to(torch.float8_e4m3fn).double())
    top = torch.tensor([0.0, 448.0, 448.1, 1.0, 3.5, 3.6, 57344.0, 1e9, 2.0 ** -20], dtype=torch.float64)
    assert O.unit_for(top).tolist() == [2.0 ** -15, 1.0, 2.0, 2.0 ** -8, 2.0 ** -7, 2.0 ** -6, 128.0, 128.0, 2.0 ** -15]


def test_bytes_that_the_scheduler_counts(monkeypatch):
    """Heads in codes of a byte with rows of 64 or 128, eight bytes of units for 64 positions and KV head, and a layer's rows as f16 for prompts."""
    import json

    from ollama_b200.models.stack import parse_stack
    from ollama_b200.models.synth import STACK_SPECS
    from ollama_b200.server.sched import predict_memory
    st = parse_stack(STACK_SPECS["vazatar-1b"])
    layers = sum(type(st.layers[r.layer].mixer).__name__ == "AttentionMixer" for r in st.runs())
    assert st.kv_bytes_per_token() == layers * 2 * 4 * 128 * 2 and st.kv_bytes_per_token(fp8=True) == layers * (2 * 4 * 128 + 1) and st.read_out_bytes() == 4 * 4 * 128
    latents = parse_stack(STACK_SPECS["kavenex-1b"])
    assert latents.kv_bytes_per_token(fp8=True) == latents.kv_bytes_per_token() and latents.read_out_bytes() == 0

    class Model:
        size = 1 << 30

        def kv(self):
            return {"general.architecture": "vazatar", "vazatar.stack": json.dumps(STACK_SPECS["vazatar-1b"])}
    for kind, dtype, each, more in (("f16", "", 2 * 4 * 128 * 2, 0), ("fp8", "", 2 * 4 * 128 + 1, 4 * 4 * 128), ("q8_0", "", 2 * 4 * 128 * 2, 0), ("fp8", "float32", 2 * 4 * 128 * 2, 0)):
        monkeypatch.setenv("OLLAMA_KV_CACHE_TYPE", kind)
        monkeypatch.setenv("B200_DTYPE", dtype)
        assert predict_memory(Model(), 4096, 3) == (1 << 30) + 3 * (layers * each * 4096 + st.state_bytes()) + more * 4096


def test_storage_of_the_paged_cache():
    from ollama_b200.engine.cache import PagedCache
    c = PagedCache(2, 100, device="cpu", fp8=True)
    a, b, d = c.add_heads(3, 64, torch.float16), c.add_heads(3, 64, torch.float32), c.add_pages(1, 96, torch.float16)
    assert isinstance(a, P.Pages8) and a.codes.shape == (4, 3, 64, 64) and b.dtype == torch.float32 and d.dtype == torch.float16
    assert isinstance(PagedCache(2, 100, device="cpu").add_heads(3, 64, torch.float16), torch.Tensor)
    c.reserve(0, 70)
    a.codes[c.owned[0][1], 1, 5] = 9
    a.unit[c.owned[0][1], 1] = 4.0
    c.copy(0, 1, 70)
    assert (a.codes[c.owned[1][1], 1, 5] == 9).all() and a.unit[c.owned[1][1], 1] == 4.0 and len(c.paged) == 4
