"""The page plan's lengths of requests that it cannot make sense of: lens is what they hold (cached), as for
every request that is not served, so that a caller who feeds lens back loses no pages."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_invalid_requests_keep_their_lengths(dtype):
    from dsv2 import _lib, ops
    _lib.device_error(clear=True)
    # new below -1, longer than its table row, a negative length, one that does not fit, and two good ones
    cached = [20, 49, -3, 40, 5, 16]
    new = [-2, 0, 1, 30, 2, 0]
    if dtype is torch.int64:
        cached[1], cached[2] = 2 ** 40, -2 ** 40
    table = torch.arange(18, dtype=torch.int32, device=DEV).view(6, 3)
    before = table.clone()
    buf = ops.page_plan_buffers(6, 64, DEV)
    ops.page_plan(cached=torch.tensor(cached, dtype=dtype, device=DEV), new=torch.tensor(new, dtype=torch.int32, device=DEV),
                  block_table=table, free_ring=torch.arange(100, 104, dtype=torch.int32, device=DEV),
                  ring_in=torch.tensor([0, 4], device=DEV), page_size=16, **buf)
    lens = buf["lens"].tolist()
    i32 = torch.iinfo(torch.int32)
    want = [min(max(c, i32.min), i32.max) for c in cached[:4]] + [7, 16]
    assert lens == want
    assert buf["counts"].tolist()[1:] == [0, 0, 4]
    assert torch.equal(table, before) and buf["ring_out"].tolist() == [0, 4]
    assert _lib.device_error(clear=True) == 2
