"""The decode engine over the paged 4-bit cache and with per-request adapters.

The 4-bit engine is compared with the bf16 engine whose cache rows are passed through the same
quantisation as they are written (so both hold the same values): what remains is the rounding of
the attention kernels, bounded like the engine's own distance to the HF model (hidden states
2e-2, logits cosine 0.999); so do adapters over the 4-bit cache.  Over the bf16 cache adapters are
compared with engines whose weights hold W + s B A, rounded to bf16: the same bounds.  (Over the
4-bit cache that comparison has no such bound: the weights' rounding moves cache elements across
rounding boundaries of the 4-bit format, by whole steps.)
"""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
LENS = [20, 33, 7, 64, 1]


def relerr(a, b):
    a, b = a.double(), b.double()
    return float((a - b).abs().max() / b.abs().max().clamp_min(1e-30))


def cosine(a, b):
    a, b = a.double(), b.double()
    return float(a @ b / (a.norm() * b.norm()))


@pytest.fixture(scope="module")
def model():
    from oracle.hf_model import build_model, dsv2_lite_config
    return build_model(dsv2_lite_config(num_layers=2), seed=3, device=torch.device(DEV), dtype=torch.bfloat16)


def prompts_of(model, lens, seed=5):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, model.config.vocab_size, (n,), generator=g) for n in lens]


def quantising_prep(ops, monkeypatch):
    """mla_prep that leaves the 4-bit cache's values in the bf16 rows it writes."""
    orig = ops.mla_prep

    def prep(*, cache, positions, cache_rows=None, **kw):
        orig(cache=cache, positions=positions, cache_rows=cache_rows, **kw)
        n = kw["q_pe_out"].shape[0]
        rows = cache_rows.long() if cache_rows is not None else torch.arange(n, device=cache.device)
        q4 = ops.latent4_cache(-(-n // 16), 16, cache.device)
        slots = torch.arange(n, device=cache.device)
        ops.latent4_write(rows=cache[rows, positions].contiguous(), slots=slots, cache=q4)
        cache[rows, positions] = ops.latent4_read(cache=q4, slots=slots, out=torch.empty(n, 576, dtype=torch.bfloat16,
                                                                                         device=cache.device))
    monkeypatch.setattr(ops, "mla_prep", prep)


@pytest.mark.parametrize("family,page,adapters", [("batch", 16, 0), ("small", 64, 0), ("batch", 48, 2), ("small", 16, 3)])
def test_int4_engine_matches_the_bf16_engine_on_the_same_cache_values(model, monkeypatch, family, page, adapters):
    from dsv2 import _lib, ops
    from dsv2.engine import DecodeEngine
    from dsv2.serving import random_adapters
    _lib.device_error(clear=True)
    prompts = prompts_of(model, LENS)
    ad = random_adapters(2, adapters, 24, len(LENS), DEV, seed=2, std=0.1) if adapters else None
    eng = DecodeEngine(model, len(LENS), 96, family, alias_hf=False, keep_logits=True, kv_format="int4", page_size=page,
                       adapters=ad)
    first = eng.prefill(prompts, max_tokens_per_chunk=50)      # chunks end inside prompts and pages
    assert eng.paged.ring.tolist()[0] == sum(-(-n // page) for n in LENS)
    traces, fed = [], []
    for _ in range(4):
        fed.append(eng.input_ids.clone())
        tr = {}
        eng.step(trace=tr)
        traces.append((tr, eng.logits.float().clone()))
    eng.plan.check()
    quantising_prep(ops, monkeypatch)
    ref = DecodeEngine(model, len(LENS), 96, family, alias_hf=False, keep_logits=True, adapters=ad)
    ref_first = ref.prefill(prompts, max_tokens_per_chunk=50)
    assert torch.equal(first, ref_first)
    for s, (tr, logits) in enumerate(traces):
        ref.input_ids.copy_(fed[s])
        rt = {}
        ref.step(trace=rt)
        for li, (a, b) in enumerate(zip(tr["hidden"], rt["hidden"])):
            assert relerr(a, b) <= 2e-2, (s, li, relerr(a, b))
        for b in range(len(LENS)):
            assert cosine(logits[b], ref.logits[b].float()) >= 0.999, (s, b)
    assert _lib.device_error(clear=True) == 0


def test_int4_graph_replay_restore_and_eager_prefill(model):
    from dsv2 import _lib
    from dsv2.engine import DecodeEngine
    prompts = prompts_of(model, LENS)
    eng = DecodeEngine(model, len(LENS), 128, "batch", alias_hf=False, kv_format="int4", page_size=16)
    eng.prefill(prompts, method="eager")
    eager = []
    for _ in range(20):                                        # rows cross page boundaries
        eng.step()
        eager.append(eng.input_ids.clone())
    taken = eng.paged.ring.tolist()
    eng.restore()
    eng.capture()
    for t in eager:
        eng.replay()
        assert torch.equal(eng.input_ids, t)
    assert eng.paged.ring.tolist() == taken                    # the same pages, taken once
    assert eng.recover() == 0
    eng.release()
    assert _lib.device_error(clear=True) == 0


def test_int4_pool_without_pages_is_reported(model):
    from dsv2.engine import DecodeEngine
    eng = DecodeEngine(model, 2, 64, "batch", alias_hf=False, kv_format="int4", page_size=16, pages=3)
    with pytest.raises(RuntimeError, match="got no pages"):
        eng.prefill(prompts_of(model, [30, 40]))
    eng.prefill(prompts_of(model, [30, 14]))                   # the pool starts over
    eng.step()
    eng.plan.check()


@pytest.mark.parametrize("family", ["batch", "small"])
def test_adapters_match_merged_weights(model, family):
    from dsv2.engine import DecodeEngine
    from dsv2.serving import random_adapters
    lens = [20, 33, 7, 12]
    prompts = prompts_of(model, lens)
    ad = random_adapters(2, 2, 16, len(lens), DEV, seed=1, std=0.1)
    ad.ids.copy_(torch.tensor([1, -1, 0, 1], dtype=torch.int32))
    ad.scales.copy_(torch.tensor([0.5, 1.5]))
    eng = DecodeEngine(model, len(lens), 64, family, alias_hf=False, keep_logits=True, adapters=ad)
    eng.prefill(prompts)
    fed = eng.input_ids.clone()
    eng.step()
    for i in (-1, 0, 1):
        rows = [r for r in range(len(lens)) if int(ad.ids[r]) == i]
        merged = copy.deepcopy(model)
        if i >= 0:
            for layer, la in zip(merged.model.layers, ad.layers):
                at = layer.self_attn
                d = (la.qkva_b[i].float() @ la.qkva_a[i].float()) * ad.scales[i]
                at.q_proj.weight.data += d[:3072].to(torch.bfloat16)
                at.kv_a_proj_with_mqa.weight.data += d[3072:].to(torch.bfloat16)
                at.o_proj.weight.data += ((la.o_b[i].float() @ la.o_a[i].float()) * ad.scales[i]).to(torch.bfloat16)
        ref = DecodeEngine(merged, len(rows), 64, family, alias_hf=False, keep_logits=True)
        ref.prefill([prompts[r] for r in rows])
        ref.input_ids.copy_(fed[rows])
        ref.step()
        for n, r in enumerate(rows):
            c = cosine(eng.logits[r].float(), ref.logits[n].float())
            assert c >= 0.999, (i, r, c)
    # the adapters do change the answer
    plain = DecodeEngine(model, len(lens), 64, family, alias_hf=False, keep_logits=True)
    plain.prefill(prompts)
    plain.input_ids.copy_(fed)
    plain.step()
    assert cosine(eng.logits[0].float(), plain.logits[0].float()) < 0.999


def test_engine_refuses_what_it_does_not_do(model):
    from dsv2.engine import DecodeEngine
    from dsv2.serving import PagedCache4, random_adapters
    with pytest.raises(ValueError):
        DecodeEngine(model, 1, 64, "batch", kv_format="int8")
    with pytest.raises(ValueError):
        PagedCache4(1, 1, 64, 24, DEV)
    with pytest.raises(ValueError):
        DecodeEngine(model, 1, 64, "batch", alias_hf=False, adapters=random_adapters(3, 1, 8, 1, DEV))
    eng = DecodeEngine(model, 1, 64, "batch", alias_hf=False, adapters=random_adapters(2, 1, 8, 1, DEV))
    with pytest.raises(NotImplementedError):
        eng.prefill(prompts_of(model, [5]), method="eager")


def test_runner_command_with_int4_cache_and_adapters(model):
    from dsv2.run import run_graph_decode
    out = run_graph_decode(model, prompts_of(model, [40])[0].to(DEV), 3, 6, "batch", dump_token_ids=True,
                           kv_cache="int4", page_size=32, lora_adapters=2, lora_rank=8)
    assert out["kv_cache"] == "int4" and len(out["generated_token_ids"]) == 3
    assert all(len(t) == 6 for t in out["generated_token_ids"])
