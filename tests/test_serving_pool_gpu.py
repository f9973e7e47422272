"""A pool that runs out of pages while the engine decodes: a request that gets no page keeps its
length and its token, writes nothing, and is reported; the other requests' pages do not change."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGE = 16
LENS = [30, 14]          # pages 2 and 1; request 0 needs its third at position 32, request 1 its second at 16


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


def engine(model, pages, family="batch", held_back=0):
    """held_back: pages of the pool that are not in the ring yet."""
    from dsv2.engine import DecodeEngine
    eng = DecodeEngine(model, len(LENS), 96, family, alias_hf=False, keep_logits=True, kv_format="int4", page_size=PAGE,
                       pages=pages)
    orig = eng.paged.reset

    def reset():
        orig()
        eng.paged.ring[1] -= held_back
    eng.paged.reset = reset
    eng.prefill(prompts_of(model, LENS))
    return eng


def run(eng, steps, replay=False, feed=None):
    """Steps of the engine; feed: the tokens that each of them is given.  Returns (fed, logits) of each."""
    out = []
    for s in range(steps):
        if feed is not None:
            eng.input_ids.copy_(torch.tensor(feed[s], device=DEV))
        fed = eng.input_ids.tolist()
        eng.replay() if replay else eng.step()
        out.append((fed, eng.logits.float().clone()))
    return out


@pytest.mark.parametrize("family", ["batch", "small"])
@pytest.mark.parametrize("replay", [False, True])
def test_requests_without_pages_wait_and_go_on(model, family, replay):
    from dsv2 import _lib
    _lib.device_error(clear=True)
    want = run(engine(model, 12, family), 8)

    def same(got, row, steps):
        for g, s in zip(got, steps):
            assert g[0][row] == want[s][0][row]
            assert cosine(g[1][row], want[s][1][row]) >= 0.999, (row, s)
    eng = engine(model, 5, family, held_back=2)           # nothing is free once the prompts have their pages
    if replay:
        eng.capture()
    got = run(eng, 2, replay, [w[0] for w in want])
    same(got, 0, [0, 1]), same(got, 1, [0, 1])
    eng.plan.check()
    eng.input_ids.copy_(torch.tensor(want[2][0], device=DEV))
    full = eng.paged.cache.clone()
    pos, ids = eng.positions.clone(), eng.input_ids.clone()
    assert pos.tolist() == [32, 16]
    for _ in range(3):                                    # both requests are at the end of their pages
        run(eng, 1, replay)
        assert torch.equal(eng.paged.cache, full)         # nobody writes into anybody's pages
        assert torch.equal(eng.positions, pos) and torch.equal(eng.input_ids, ids)
        assert eng.next_ids.tolist() == [-1, -1]
        with pytest.raises(RuntimeError, match="got no pages"):
            eng.plan.check()
    eng.paged.ring[1] += 1                                # a page comes back: the first request goes on
    held = eng.paged.block_table[1, 0].item()
    of_one = eng.paged.cache[:, held].clone()
    same(run(eng, 3, replay, [[want[s][0][0], int(ids[1])] for s in (2, 3, 4)]), 0, [2, 3, 4])
    assert torch.equal(eng.paged.cache[:, held], of_one)
    assert eng.positions.tolist() == [35, 16] and int(eng.input_ids[1]) == int(ids[1])
    eng.paged.ring[1] += 1                                # and another: so does the second
    got = run(eng, 3, replay, [[want[a][0][0], want[b][0][1]] for a, b in ((5, 2), (6, 3), (7, 4))])
    same(got, 0, [5, 6, 7]), same(got, 1, [2, 3, 4])
    assert eng.positions.tolist() == [38, 19]
    assert int(eng.plan.buf["counts"][3]) == 0
    with pytest.raises(RuntimeError, match="got no pages"):   # steps that serve everybody again do not hide the others
        eng.plan.check()
    eng.plan.clear()
    eng.plan.check()
    eng.release()
    assert _lib.device_error(clear=True) == 0


def test_a_new_prefill_and_restore_forget_missed_steps(model):
    eng = engine(model, 3)
    run(eng, 3)
    with pytest.raises(RuntimeError, match="got no pages"):
        eng.plan.check()
    eng.restore()
    eng.plan.check()
    first = [g[0] for g in run(eng, 3)]
    eng.prefill(prompts_of(model, LENS))
    eng.plan.check()
    assert [g[0] for g in run(eng, 3)] == first


def test_table_entries_that_were_never_given_name_no_page(model):
    from dsv2.serving import PagedCache4
    eng = engine(model, 12)
    held = [-(-n // PAGE) for n in LENS]
    for r, h in enumerate(held):
        assert bool((eng.paged.block_table[r, h:] == -1).all())
    c = PagedCache4(1, 3, 64, 16, DEV)
    assert bool((c.block_table == -1).all())


@pytest.mark.parametrize("family,V,T", [("small", 3001, 3), ("batch", 5000, 33)])
def test_lm_head_advances_served_rows_alone(family, V, T):
    from dsv2 import ops
    g = torch.Generator().manual_seed(T)
    w = (torch.randn(V, 2048, generator=g) * 0.02).to(torch.bfloat16).to(DEV)
    x = torch.randn(T, 2048, generator=g).to(torch.bfloat16).to(DEV)
    f = ops.FAMILY_SMALL if family == "small" else ops.FAMILY_BATCH

    def head(**kw):
        t = {"next_ids": torch.full((T,), -7, dtype=torch.int64, device=DEV),
             "input_ids": torch.arange(T, device=DEV) + 100, "positions": torch.arange(T, device=DEV) * 3}
        ops.lm_head_argmax(w=w, x=x, keys=torch.zeros(((V + 15) // 16) * T, dtype=torch.int64, device=DEV), family=f, **t, **kw)
        return t
    want = head()
    served = torch.arange(T, device=DEV) * 5
    served[::3] = -1
    missed = torch.full((1,), 4, dtype=torch.int32, device=DEV)
    got = head(served=served, missed=missed)
    live = served >= 0
    for k, idle in (("next_ids", torch.full((T,), -1, device=DEV)), ("input_ids", torch.arange(T, device=DEV) + 100),
                    ("positions", torch.arange(T, device=DEV) * 3)):
        assert torch.equal(got[k], torch.where(live, want[k], idle)), k
    assert int(missed) == 4 + int((~live).sum())
    with pytest.raises(ValueError):
        head(served=served[:-1], missed=missed)
    with pytest.raises(ValueError):
        head(served=served)
