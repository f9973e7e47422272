"""Operands of the serving operators on another GPU, of another type or too small are refused before the
library is called.  No GPU is needed: CPU tensors that say they are on a device, and a library that notes the
call."""
import pytest
import torch

from dsv2 import _lib, ops


class On(torch.Tensor):
    """A CPU tensor that calls itself a tensor of GPU `gpu`."""
    gpu = 0

    def get_device(self):
        return self.gpu

    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", self.gpu))


def on(t, gpu=0):
    r = t.as_subclass(On)
    r.gpu = gpu
    return r


@pytest.fixture
def calls(monkeypatch):
    out = []
    monkeypatch.setattr(_lib, "call", lambda name, *args: out.append(name))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: 0, raising=False)
    return out


def z(*shape, dtype=torch.bfloat16):
    return on(torch.zeros(shape, dtype=dtype))


def i32(*shape):
    return z(*shape, dtype=torch.int32)


def i64(*shape):
    return z(*shape, dtype=torch.int64)


def f32(*shape):
    return z(*shape, dtype=torch.float32)


def plan():
    return ops.page_plan, dict(cached=i64(3), new=i32(3), block_table=i32(3, 4), free_ring=i32(9), ring_in=i64(2), page_size=16,
                               ring_out=i64(2), token_row=i32(5), positions=i64(5), slots=i64(5), cu_new=i32(4), lens=i32(3),
                               counts=i32(4), sync=i32(1))


def write():
    return ops.latent4_write, dict(rows=z(3, 576), slots=i64(3), cache=z(2, 6400, dtype=torch.uint8))


def read():
    return ops.latent4_read, dict(out=z(3, 576), slots=i64(3), cache=z(2, 6400, dtype=torch.uint8))


def attention():
    return ops.mla_decode_q4, dict(q_abs=z(3, 16, 512), q_pe=z(3, 16, 64), cache=z(2, 6400, dtype=torch.uint8), block_table=i32(3, 4),
                                   positions=i64(3), page_size=16, softmax_scale=1.0, o_lat=z(3, 16, 512), o_part=f32(4, 16, 512),
                                   ml_part=f32(4, 16, 2), cuts=i32(2, 4), seq_rows=i32(3))


def adapters():
    return ops.lora, dict(x=z(3, 64), a=z(2, 8, 64), b=z(2, 16, 8), ids=i32(3), ranks=i32(2), scales=f32(2), y=z(3, 16), low=f32(24),
                          order=i32(9), base=f32(2, 3, 16), token_row=i32(3))


def projection():
    return ops.lora_linear, dict(x=z(3, 64), w=z(16, 64), a=z(2, 8, 64), b=z(2, 16, 8), ids=i32(3), ranks=i32(2), scales=f32(2),
                                 y=z(3, 16), parts=f32(1, 3, 16), low=f32(24), order=i32(9), xs=z(3, 64), lists=i32(1, 514))


@pytest.mark.parametrize("make", [plan, write, read, attention, adapters, projection])
def test_operands_on_another_gpu_are_refused(calls, monkeypatch, make):
    f, kw = make()
    f(**kw)
    assert len(calls) == 1
    for name, t in kw.items():
        if isinstance(t, torch.Tensor):
            with pytest.raises(ValueError):
                f(**dict(kw, **{name: on(t.as_subclass(torch.Tensor), 1)}))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(ValueError):
        f(**kw)
    assert len(calls) == 1


def prep():
    return ops.mla_prep_q4, dict(qkva=f32(2, 3, 3648), kv_norm_w=z(512), eps=1e-6, cos=f32(9, 32), sin=f32(9, 32), positions=i64(3),
                                 slots=i64(3), cache=z(2, 6400, dtype=torch.uint8), q_pe_out=z(3, 16, 64), q_nope_out=z(3, 16, 128))


@pytest.mark.parametrize("name,bad", [
    ("positions", i32(3)), ("positions", i64(6)[::2]), ("positions", i64(4)), ("slots", i64(2)), ("slots", i32(3)),
    ("kv_norm_w", f32(512)), ("kv_norm_w", z(511)), ("q_pe_out", f32(3, 16, 64)), ("q_pe_out", z(2, 16, 64)), ("q_nope_out", z(2, 16, 128)),
    ("sin", f32(8, 32)), ("sin", f32(9, 64)[:, :32]), ("cos", f32(9, 31)), ("cache", z(6399, dtype=torch.uint8))])
def test_prep_refuses_operands_that_the_kernel_would_read_past(calls, name, bad):
    f, kw = prep()
    f(**kw)
    assert len(calls) == 1
    if name == "cos":
        kw["sin"] = bad
    with pytest.raises((ValueError, NotImplementedError)):
        f(**dict(kw, **{name: bad}))
    assert len(calls) == 1


def test_prep_refuses_operands_on_another_gpu(calls):
    f, kw = prep()
    for name, t in kw.items():
        if isinstance(t, torch.Tensor):
            with pytest.raises(ValueError):
                f(**dict(kw, **{name: on(t.as_subclass(torch.Tensor), 1)}))
    assert not calls
