"""CPU tests of the paged 4-bit serving operators: the format's arithmetic, the sequential page
plan, and the refusals of the entry points (which come before any CUDA call)."""
import ctypes

import pytest
import torch

from oracle import serving as S


def test_scales_and_values_are_exact_in_bf16_and_fp16():
    v = torch.arange(-8, 8).double()
    x = (S.SCALES[:, None] * v).view(-1)
    assert torch.equal(x.to(torch.bfloat16).double(), x)
    assert torch.equal(x.to(torch.float16).double(), x)
    code = torch.arange(S.MAX_CODE + 1)
    assert torch.equal((code << 7).to(torch.int16).view(torch.float16).double(), S.SCALES)


def test_quantisation_error_is_at_most_half_a_step():
    g = torch.Generator().manual_seed(0)
    rows = (torch.randn(200, 576, generator=g) * torch.exp(2 * torch.randn(200, 1, generator=g))).to(torch.bfloat16)
    val = S.values(rows)[:, :512].view(-1, 16, 32)
    x = rows[:, :512].double().view(-1, 16, 32)
    _, code = S.quantise(rows)
    step = S.scale_value(code)[..., None]
    fits = x.abs().amax(-1) <= 7 * 60                     # larger groups saturate
    val, x, step = val[fits], x[fits], step[fits]
    # the scale is within 1/16 of max / 7, so the largest element is at most 7.5 steps: it may
    # lose half a step to the clamp at 7 as well
    assert float(((val - x).abs() / step).max()) <= 0.5 + 2 ** -4


def test_layout_places_every_byte_once():
    rows = torch.zeros(16, 576, dtype=torch.bfloat16)
    _, off = S.token_bytes(rows, torch.arange(16))
    assert torch.equal(off.view(-1).sort().values, torch.arange(6400))


def test_fragment_reads_hit_all_banks():
    """The shared-memory reads the layout is made for: one wavefront per 128 bytes."""
    def f(p):
        return 2 * (p & 1) + 4 * (((p >> 1) ^ (p >> 2)) & 1)
    # scores: 8 lanes read 16 bytes: tokens p, p + 4, four neighbouring groups
    for p in (0, 1, 2, 3, 8, 9, 10, 11):
        for c0 in (0, 4, 8, 12):
            at = {((256 * t + 16 * ((c0 + i) ^ f(t))) // 16) % 8 for t in (p, p + 4) for i in range(4)}
            assert len(at) == 8
            at = {((128 * t + 16 * ((h + i) ^ (t & 4))) // 16) % 8 for h in (0,) for t in (p, p + 4) for i in range(4)}
            assert len(at) == 8
    # P V: 32 lanes read a word: tokens with p & 3 = 0..3, two neighbouring groups of four words
    for base in (0, 4, 8, 12):
        for c0 in range(0, 16, 2):
            at = {((256 * (base + t) + 16 * ((c0 + i) ^ f(base + t)) + 4 * w) // 4) % 32
                  for t in range(4) for i in range(2) for w in range(4)}
            assert len(at) == 32


def test_sequential_plan_small_case():
    table = [[4, -1, -1], [9, 2, -1], [7, -1, -1]]
    ring = [11, 12, 13, 14]
    out = S.page_plan([16, 20, 3], [1, -1, 14], table, ring, (2, 4), 16, 20)
    assert table == [[4, 13, -1], [9, 2, -1], [7, 14, -1]]
    assert ring == [9, 2, 13, 14] and out["ring_out"] == [4, 6] and out["lens"] == [17, 0, 17]
    assert out["slots"][:3] == [13 * 16, 7 * 16 + 3, 7 * 16 + 4] and out["slots"][14] == 14 * 16
    assert out["token_row"][15:] == [-1] * 5 and out["counts"] == [15, 2, 2, 0]


def _call(name, *args):
    from dsv2 import _lib
    _lib.call(name, *args)


def test_page_plan_refusals():
    from dsv2 import _lib

    def args(**kw):
        a = _lib.PagePlanArgs(*([4096] * 13), 4, 8, 2, 4, 16, 8, 0)
        a.lens = 8192
        for k, v in kw.items():
            setattr(a, k, v)
        return ctypes.byref(a), None
    for kw in (dict(block_table=None), dict(cached=None), dict(slots=None), dict(page_size=0), dict(page_size=24),
               dict(width=0), dict(table_stride=3), dict(ring_size=0), dict(requests=-1), dict(token_capacity=-1),
               dict(lens=4096), dict(sync=None)):
        with pytest.raises(ValueError):
            _call("dsv2_page_plan", *args(**kw))
    with pytest.raises(NotImplementedError):
        _call("dsv2_page_plan", *args(width=1 << 28, table_stride=1 << 28))


def test_latent4_refusals():
    for rows, stride, slots, n, cache, blocks in ((None, 576, 16, 1, 16, 1), (16, 570, 16, 1, 16, 1), (16, 580, 16, 1, 16, 1),
                                                  (8, 576, 16, 1, 16, 1), (16, 576, None, 1, 16, 1), (16, 576, 16, -1, 16, 1),
                                                  (16, 576, 16, 1, 24, 1), (16, 576, 16, 1, 16, 0)):
        with pytest.raises(ValueError):
            _call("dsv2_latent4_write", rows, stride, slots, n, cache, blocks, None)
        with pytest.raises(ValueError):
            _call("dsv2_latent4_read", cache, blocks, slots, n, rows, stride, None)
    with pytest.raises(NotImplementedError):
        _call("dsv2_latent4_write", 16, 576, 16, 1 << 40, 16, 1, None)
    from dsv2 import _lib
    with pytest.raises(ValueError):
        _call("dsv2_mla_prep_q4", ctypes.byref(_lib.MlaPrepArgs()), None, 1, 16, None)
    with pytest.raises(ValueError):
        _call("dsv2_mla_prep_q4", ctypes.byref(_lib.MlaPrepArgs()), 16, 1, 16, None)


def test_lora_refusals():
    from dsv2 import _lib

    def args(**kw):
        a = _lib.LoraArgs(4096, 64, 4096, 4096, 4096, None, 4096, 4096, None, 0, None, 0, 0, 4096, None, 4096, 16, 1, 0, 0, 3, 2, 8, 3, 64, 16)
        for k, v in kw.items():
            setattr(a, k, v)
        return ctypes.byref(a), None
    for kw in (dict(x=None), dict(y=None), dict(a=None), dict(low=None), dict(n_base=1), dict(ids_len=2), dict(x=4104),
               dict(x_row_stride=60), dict(y_row_stride=20), dict(tokens=-1), dict(adapters=-1), dict(low_parts=0), dict(w=4096),
               dict(tokens=17, ids_len=17)):
        with pytest.raises(ValueError):
            _call("dsv2_lora", *args(**kw))
    for kw in (dict(k=60), dict(n=12), dict(rank=4), dict(rank=136), dict(y_dtype=1)):
        with pytest.raises(NotImplementedError):
            _call("dsv2_lora", *args(**kw))


def test_python_wrappers_refuse_cpu_tensors_and_wrong_shapes():
    from dsv2 import ops
    z = torch.zeros
    with pytest.raises(NotImplementedError):
        ops.latent4_write(rows=z(2, 576, dtype=torch.bfloat16), slots=z(2, dtype=torch.int64), cache=z(1, 6400, dtype=torch.uint8))
    with pytest.raises(NotImplementedError):
        ops.page_plan(cached=z(1, dtype=torch.int32), new=z(1, dtype=torch.int32), block_table=z(1, 2, dtype=torch.int32),
                      free_ring=z(4, dtype=torch.int32), ring_in=z(2, dtype=torch.int64), page_size=16,
                      **ops.page_plan_buffers(1, 1, "cpu"))
    with pytest.raises(ValueError):
        ops.latent4_cache(4, 24, "cpu")
    with pytest.raises(ValueError):
        ops.mla_decode_q4(q_abs=z(2, 16, 500, dtype=torch.bfloat16), q_pe=z(2, 16, 64, dtype=torch.bfloat16),
                          cache=z(1, 6400, dtype=torch.uint8), block_table=z(2, 1, dtype=torch.int32),
                          positions=z(2, dtype=torch.int64), page_size=16, softmax_scale=1.0,
                          o_lat=z(2, 16, 500, dtype=torch.bfloat16), **_ws(ops))
    with pytest.raises(NotImplementedError):
        ops.lora(x=z(2, 64, dtype=torch.bfloat16), a=z(1, 8, 64, dtype=torch.bfloat16), b=z(1, 16, 8, dtype=torch.bfloat16),
                 ids=z(2, dtype=torch.int32), ranks=z(1, dtype=torch.int32), scales=z(1), y=z(2, 16), low=z(16))
    assert ops.latent4_cache(3, 32, "cpu", layers=2).shape == (2, 3, 12800)


def _ws(ops):
    return {"o_part": torch.zeros(2, 16, 512), "ml_part": torch.zeros(2, 16, 2), "cuts": torch.zeros(1, 4, dtype=torch.int32)}
