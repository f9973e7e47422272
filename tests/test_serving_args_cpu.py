"""Refusals of the serving entry points that come before any CUDA call."""
import pytest


def test_lm_head_served_refusals():
    from dsv2 import _lib

    def call(served=4096, missed=4096, positions=4096, numel=2, w=4096):
        _lib.call("dsv2_lm_head_argmax_served", w, 32, 64, 4096, 64, 2, 4096, 100, 4096, 4096, positions, numel, None, served, missed,
                  1, None)
    for kw in (dict(served=None), dict(missed=None), dict(numel=1), dict(numel=3), dict(w=None)):
        with pytest.raises(ValueError):
            call(**kw)


def test_lora_refuses_a_k_that_its_projection_cannot_take():
    """Above 16 tokens, or with the projection in several pieces of k, the projection is dsv2_linear's: k % 64."""
    import ctypes

    from dsv2 import _lib

    def call(**kw):
        a = _lib.LoraArgs()
        for name in ("x", "a", "b", "ids", "ranks", "scales", "w", "base", "low", "order", "y"):
            setattr(a, name, 4096)
        for name, v in dict(x_row_stride=72, w_row_stride=72, base_row_stride=16, y_row_stride=16, low_parts=1, n_base=1, ids_len=64,
                            adapters=2, rank=8, k=72, n=16).items():
            setattr(a, name, v)
        for name, v in kw.items():
            setattr(a, name, v)
        _lib.call("dsv2_lora", ctypes.byref(a), None)
    for kw in (dict(tokens=17), dict(tokens=16, n_base=2), dict(tokens=40, ids_len=40)):
        with pytest.raises(NotImplementedError, match="multiple of 64"):
            call(**kw)
