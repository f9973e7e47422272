"""Engines with adapters over more than 256 token rows: kernel prefill of long prompts, and a decode batch of the
small family, whose projections and adapters are then one GEMM.  Same bounds as the engine's other comparisons (logits
cosine 0.999)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def model():
    from oracle.hf_model import build_model, dsv2_lite_config
    return build_model(dsv2_lite_config(num_layers=2), seed=3, device=torch.device(DEV), dtype=torch.bfloat16)


def prompts_of(model, lens, seed=5):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, model.config.vocab_size, (n,), generator=g) for n in lens]


def cosine(a, b):
    a, b = a.double(), b.double()
    return float(a @ b / (a.norm() * b.norm()))


@pytest.mark.parametrize("kv", ["bf16", "int4"])
def test_prefill_in_one_chunk_and_in_short_ones(model, kv):
    """Chunks of 613 tokens against chunks of at most 100 (whose adapters take the short runs' kernels): the tokens after the prompts
    see the same context."""
    from dsv2 import _lib
    from dsv2.engine import DecodeEngine
    from dsv2.serving import random_adapters
    _lib.device_error(clear=True)
    lens = [301, 7, 250, 55]
    logits = []
    fed = None
    for chunk in (4096, 100):
        ad = random_adapters(2, 3, 24, len(lens), DEV, seed=2, std=0.1)
        eng = DecodeEngine(model, len(lens), 320, "batch", alias_hf=False, keep_logits=True, kv_format=kv, page_size=32, adapters=ad)
        eng.prefill(prompts_of(model, lens), max_tokens_per_chunk=chunk)
        if fed is None:
            fed = eng.input_ids.clone()
        eng.input_ids.copy_(fed)
        eng.step()
        logits.append(eng.logits.float().clone())
    for b in range(len(lens)):
        assert cosine(logits[0][b], logits[1][b]) >= 0.999, b
    assert _lib.device_error(clear=True) == 0


def test_small_family_of_many_rows_matches_the_batch_family(model):
    from dsv2 import _lib
    from dsv2.engine import DecodeEngine
    from dsv2.serving import random_adapters
    _lib.device_error(clear=True)
    B = 260
    prompts = prompts_of(model, [2 + i % 3 for i in range(B)])
    logits = []
    fed = None
    for family in ("batch", "small"):
        ad = random_adapters(2, 3, 24, B, DEV, seed=2, std=0.1)
        eng = DecodeEngine(model, B, 32, family, alias_hf=False, keep_logits=True, adapters=ad)
        eng.prefill(prompts)
        if fed is None:
            fed = eng.input_ids.clone()
        eng.input_ids.copy_(fed)
        eng.step()
        logits.append(eng.logits.float().clone())
    for b in range(0, B, 7):
        assert cosine(logits[0][b], logits[1][b]) >= 0.999, b
    assert _lib.device_error(clear=True) == 0
