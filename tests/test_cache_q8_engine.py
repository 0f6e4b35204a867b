"""Engines whose cache is kept in 8 bits: logits against the plain model with quantised keys and values, under every way of cutting
the work, for every architecture; requests served, graphs, commands."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import divitar_helpers
import figotar_helpers
import fororax_helpers
import plain_gpt
import plain_q8
import tiny_configs as tc
import vatevik_helpers
import vekedra_helpers
import vipovik_helpers

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OTHERS = {"Vekedra": vekedra_helpers.MIXED, "Figotar": figotar_helpers.MIXED, "Vatevik": vatevik_helpers.MIXED, "Divitar": divitar_helpers.MIXED,
          "Fororax": fororax_helpers.MIXED, "Vipovik": vipovik_helpers.MIXED}


def coded_attention(h, c_attn_w, c_attn_b, c_proj_w, c_proj_b, n_head):
    """``plain_gpt.attention`` with keys and values as an 8-bit cache holds them."""
    T, d = h.shape
    q, k, v = (x.reshape(T, n_head, d // n_head) for x in (h @ c_attn_w + c_attn_b).split(d, dim=1))
    out = torch.zeros(T, n_head, d // n_head, dtype=h.dtype)
    held = []
    for x in (k, v):
        codes, scale = plain_q8.quantise(x)
        held.append(codes * scale.double()[..., None])
    for p in range(T):
        for i in range(n_head):
            out[p, i] = plain_q8.attend(q[p, i], held[0][:, i], held[1][:, i], p, list(range(p + 1)), (d // n_head) ** -0.5)[0]
    return out.reshape(T, d) @ c_proj_w + c_proj_b


def plain_logits(folder, tokens, monkeypatch):
    cfg, w = plain_gpt.read_model_folder(folder, torch.float64)
    exact = plain_gpt.forward(cfg, w, tokens)
    with monkeypatch.context() as m:
        m.setattr(plain_gpt, "attention", coded_attention)
        return exact, plain_gpt.forward(cfg, w, tokens)


def run_in(eng, tokens, portions):
    """Every row's logits of a text run in portions of the given sizes (the last one repeated)."""
    from cbis_b200.engine import StepEntry
    slot = eng.open_request(0)
    out, at = [], 0
    while at < len(tokens):
        n = min(portions[min(len(out), len(portions) - 1)], len(tokens) - at)
        out.append(eng.forward_step([StepEntry(slot, at, tokens[at:at + n], list(range(n)))]).double().cpu())
        at += n
    eng.close_request(slot)
    return torch.cat(out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_logits_against_the_plain_model(tiny, dtype, monkeypatch):
    """A 32-bit engine agrees with the plain model of quantised keys and values far better than with the exact one: what is left are
    codes that 32-bit sums put on the other side of a half step (one of some ten thousand, a step each, where every code is off by
    a quarter step on average)."""
    import cbis_b200 as cb
    folder, cfg, page = tiny
    g = torch.Generator().manual_seed(5)
    tokens = torch.randint(0, cfg["vocab_size"], (61,), generator=g).tolist()
    exact, coded = plain_logits(folder, tokens, monkeypatch)
    moved = (coded - exact).abs().max().item()
    assert moved > 0
    eng = cb.Engine(folder, dtype=dtype, page_size=page, num_pages=40, max_num_seqs=3, max_batched_tokens=64, cache_dtype="int8")
    for portions in ([61], [1], [16], [7, 1, 20, 1, 1, 31]):
        off = (run_in(eng, tokens, portions) - coded).abs().max().item()
        assert off <= (0.15 * moved if dtype == "float32" else 0.03 * coded.abs().max().item()), portions


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(OTHERS))
def test_every_architecture(name):
    """Logits near those of the cache in the model's type (8 bits change a key by half a 127th of its largest number at most), and the
    same however the text is cut.

    In 32 bits the distance q is the codes' alone.  In bfloat16 the two engines' logits are (coded 16 - coded 32) + (coded 32 - full 32) +
    (full 32 - full 16) apart: q, and twice what bfloat16 does to a model's logits, b (of the full cache); once more b for the
    values that are rounded as they are read back.  Two cuts in bfloat16 differ by the roundings of two runs, 2 b, and what these
    move across a code's border, which is less than q."""
    import cbis_b200 as cb
    cfg = OTHERS[name]
    opts = dict(seed=3, page_size=16, num_pages=24, max_num_seqs=2, max_batched_tokens=64, max_model_len=256)
    tokens = torch.randint(0, cfg["vocab"], (150,), generator=torch.Generator().manual_seed(1)).tolist()
    far = lambda x, y: (x - y).pow(2).mean().sqrt().item()      # noqa: E731
    full, one, cuts = {}, {}, {}
    for dtype in ("float32", "bfloat16"):
        full[dtype] = run_in(cb.Engine.from_random(cfg, dtype=dtype, **opts), tokens, [64])
        eng = cb.Engine.from_random(cfg, dtype=dtype, cache_dtype="int8", **opts)
        one[dtype] = run_in(eng, tokens, [64])
        assert torch.isfinite(one[dtype]).all()
        cuts[dtype] = [run_in(eng, tokens, portions) for portions in ([50, 1, 1, 40, 1, 57], [1])]
    size = full["float32"].pow(2).mean().sqrt().item()
    q, b = far(one["float32"], full["float32"]), far(full["bfloat16"], full["float32"])
    assert 0 < q < 0.1 * size
    assert far(one["bfloat16"], full["bfloat16"]) < q + 3 * b
    for cut in cuts["float32"]:
        assert far(cut, one["float32"]) < 0.25 * q
    for cut in cuts["bfloat16"]:
        assert far(cut, one["bfloat16"]) < q + 2 * b


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,hd,window", [(4, 4, 64, 0), (8, 2, 128, 0), (4, 1, 32, 40), (2, 2, 256, 0), (4, 2, 24, 30)])
def test_head_sizes_and_windows(heads, kv_heads, hd, window):
    """The built-in attention at the sizes of every path: prompts long enough for the read back, decoded tokens, windows."""
    import cbis_b200 as cb
    from cbis_b200.config import LayerSpec, ModelSpec, PartSpec

    class Config:
        @staticmethod
        def model_spec():
            w = heads * hd
            att = PartSpec("attention", {"width": w, "n_head": heads, "n_kv_head": kv_heads, "head_dim": hd, "scale": hd ** -0.5, "window": window})
            norm, ffn = PartSpec("layernorm", {"width": w, "eps": 1e-5}), PartSpec("dense", {"width": w, "inner": 64, "activation": "gelu_erf"})
            layers = (LayerSpec("h.0.", "pre_norm", att, ffn, norm, norm), LayerSpec("h.1.", "pre_norm", att, ffn, norm, norm),
                      LayerSpec("h.2.", "pre_norm", att, ffn, norm, norm, cache_source=0))      # reads the first layer's cache
            return ModelSpec(w, 101, 400, "wte.weight", PartSpec("learned", {"width": w, "n_positions": 400}), layers, (0, 1, 2), norm, "ln_f.", None)

    tokens = torch.randint(0, 101, (330,), generator=torch.Generator().manual_seed(2)).tolist()
    for dtype in ("float32", "bfloat16"):
        opts = dict(seed=1, dtype=dtype, page_size=16, num_pages=30, max_num_seqs=2, max_batched_tokens=256)
        full = run_in(cb.Engine.from_random(Config(), **opts), tokens, [200, 90, 1])
        eng = cb.Engine.from_random(Config(), cache_dtype="int8", **opts)
        one, cut = run_in(eng, tokens, [200, 90, 1]), run_in(eng, tokens, [3, 60, 1, 5, 256])
        rms = (one - full).pow(2).mean().sqrt().item()
        assert 0 < rms < 0.05 * full.pow(2).mean().sqrt().item()
        assert (cut - one).pow(2).mean().sqrt().item() < (0.25 * rms if dtype == "float32" else 2 * rms)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,pages", [("float32", 14), ("bfloat16", 14), ("float32", 8), ("bfloat16", 8)])
def test_requests_served(folder_a, dtype, pages, monkeypatch):
    """Continuous batching with preemption, freed pages filled with NaN, graphs captured ahead: every request's tokens are those that it
    gets alone."""
    import cbis_b200 as cb
    g = torch.Generator().manual_seed(9)
    prompts = [torch.randint(0, tc.TINY_A["vocab_size"], (n,), generator=g).tolist() for n in (5, 17, 33, 40, 2, 61)]
    opts = dict(dtype=dtype, page_size=tc.PAGE_A, max_batched_tokens=48, cache_dtype="int8")
    eng = cb.Engine(folder_a, num_pages=pages, max_num_seqs=4, prefill_chunk=16, poison_freed_pages=True, **opts)
    eng.warm_up()
    outs = eng.generate(prompts, cb.SamplingParams(max_new_tokens=20))
    assert (eng.scheduler.preemptions() > 0) == (pages == 8) and eng.runner.graph_replays > 0 and eng.pages_poisoned > 0
    assert eng.pool.manager.free_pages(0) == pages and eng.pool.manager.check() == ""
    solo = cb.Engine(folder_a, num_pages=40, max_num_seqs=1, **opts)
    cfg, w = plain_gpt.read_model_folder(folder_a, torch.float64)
    monkeypatch.setattr(plain_gpt, "attention", coded_attention)
    for p, o in zip(prompts, outs):
        if dtype == "float32":
            assert solo.generate([p], cb.SamplingParams(max_new_tokens=20))[0] == o
        logits = plain_gpt.forward(cfg, w, p + o[:-1])
        for j, t in enumerate(o):      # every token is, by the plain model of quantised keys and values, within a margin of the best
            row = logits[len(p) - 1 + j]
            assert row[t] >= row.max() - (0.005 if dtype == "float32" else 0.03) * logits.abs().max()


@pytest.mark.gpu
def test_a_step_replayed_and_a_loop_on_the_device(folder_a):
    """Decode steps as graphs, and many of them without the host, store and read the same codes as steps launch by launch."""
    import cbis_b200 as cb
    from cbis_b200.engine import StepEntry
    prompts = [[3, 1, 4, 1, 5], list(range(30, 60))]
    tokens = []
    for graphs in (False, True):
        eng = cb.Engine(folder_a, dtype="bfloat16", page_size=tc.PAGE_A, num_pages=24, max_num_seqs=2, max_batched_tokens=64, cache_dtype="int8")
        eng.runner.use_graphs = graphs
        tokens.append(eng.generate(prompts, cb.SamplingParams(max_new_tokens=24)))
    assert tokens[0] == tokens[1]
    eng = cb.Engine(folder_a, dtype="bfloat16", page_size=tc.PAGE_A, num_pages=24, max_num_seqs=2, max_batched_tokens=64, cache_dtype="int8")
    slots = [eng.open_request(i) for i in range(2)]
    first = [int(eng.forward_step([StepEntry(s, 0, p, [len(p) - 1])]).argmax()) for s, p in zip(slots, prompts)]
    for s in slots:
        assert eng.pool.manager.append(s, 12)
    loop = eng.runner.decode_loop([StepEntry(s, len(p), [t], [0]) for s, p, t in zip(slots, prompts, first)])
    seen = [loop.last_tokens()]
    for _ in range(8):
        loop.run(1)
        seen.append(loop.last_tokens())
    assert [[f] + [s[i] for s in seen] for i, f in enumerate(first)] == [t[:10] for t in tokens[0]]


@pytest.mark.gpu
def test_memory(folder_a):
    import cbis_b200 as cb
    opts = dict(page_size=16, num_pages=12, max_num_seqs=2, max_batched_tokens=32)
    for dtype, size in (("bfloat16", 2), ("float32", 4)):
        full, coded = cb.Engine(folder_a, dtype=dtype, **opts).pool, cb.Engine(folder_a, dtype=dtype, cache_dtype="int8", **opts).pool
        layers, heads, hd = tc.TINY_A["n_layer"], tc.TINY_A["n_head"], tc.TINY_A["n_embd"] // tc.TINY_A["n_head"]
        assert full.bytes_per_token() == layers * 2 * heads * hd * size
        assert coded.bytes_per_token() == layers * 2 * heads * (hd + 4)
        kept = sum(g.storage.numel() + 4 * g.scale_storage.numel() for g in coded.groups)
        assert kept >= coded.bytes_per_token() * 12 * 16 and coded.layer_cache[0].values is coded.layer_cache[1].values
        assert all(t.data_ptr() % 256 == 0 for lc in coded.layer_cache.values() for t in lc.arrays.values())
    by_memory = cb.Engine(folder_a, dtype="bfloat16", page_size=16, max_num_seqs=2, max_batched_tokens=32, cache_dtype="int8").pool
    assert by_memory.groups[0].num_pages == 2 * (tc.TINY_A["n_positions"] // 16)


@pytest.mark.gpu
def test_command_line(folder_a):
    run = [sys.executable, os.path.join(ROOT, "bin", "generate"), folder_a, "--prompt-ids", "1,2,3,4,5", "--max-new-tokens", "9", "--json", "--dtype", "float32"]
    import cbis_b200 as cb
    eng = cb.Engine(folder_a, dtype="float32", cache_dtype="int8", num_pages=8)
    want = eng.generate([[1, 2, 3, 4, 5]], cb.SamplingParams(max_new_tokens=9))[0]
    out = subprocess.run(run + ["--cache-dtype", "int8"], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    assert json.loads(out.stdout)["tokens"] == want


@pytest.mark.gpu
def test_what_cannot_be_kept_in_8_bits_is_refused(folder_a):
    import cbis_b200 as cb
    with pytest.raises(ValueError, match="cache_dtype 'int4'"):
        cb.Engine(folder_a, cache_dtype="int4")


def test_a_mixer_that_reads_its_pages_itself_is_refused():
    from types import SimpleNamespace
    from cbis_b200.cache.pool import refuse_coded
    from cbis_b200.parts import CacheArray, CacheNeed, Mixer
    from cbis_b200.parts.attention import PagedAttention

    class Own(Mixer):
        def cache_need(self):
            return CacheNeed((CacheArray("latent", 1, 10),))

    layer = lambda m, src=None: SimpleNamespace(mixer=m, spec=SimpleNamespace(cache_source=src))      # noqa: E731
    fine = PagedAttention(64, 2, 2, 32, 1.0)
    refuse_coded(SimpleNamespace(layers=[layer(fine), layer(PagedAttention(64, 2, 2, 32, 1.0, own_kv=False), 0)]))
    with pytest.raises(ValueError, match="layer 1: Own"):
        refuse_coded(SimpleNamespace(layers=[layer(fine), layer(Own())]))


def test_bytes_of_a_page():
    from cbis_b200.cache.pool import CacheGroup
    from cbis_b200.parts import CacheNeed
    g = CacheGroup(CacheNeed.keys_values(3, 40), [0, 2], 8, 0)
    assert g.bytes_per_page(2) == 2 * 2 * 3 * 40 * 8 * 2
    assert g.bytes_per_page(2, True) == 2 * 2 * 3 * (40 + 4) * 8
    assert np.isclose(g.bytes_per_page(4, True) / g.bytes_per_page(4), 44 / 160)
