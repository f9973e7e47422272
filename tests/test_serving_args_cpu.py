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
